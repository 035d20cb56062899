"""The tensor IR: an SSA node list with shapes inferred at creation.

Host-side restatement of the reference's IR so the backend can be driven
without a JavaScript engine.  Semantics follow ``src/ir/graph.js`` (builder,
``emit``, composites) and ``src/ir/shapes.js`` (shape rules, broadcasting).
Node ids are list positions, so a graph is always in topological order.

Interchange is the reference's ``Graph.toJSON`` form
(``{"nodes": [{op, inputs, attrs, shape}]}``, src/ir/graph.js:48-50), so
graphs written by the reference (golden/cases.json) load unchanged.
"""
from __future__ import annotations

import copy
import math

UNARY = ("neg", "exp", "log", "relu", "tanh", "step", "stopGradient", "sqrt")
BINARY = ("add", "sub", "mul", "div")
REDUCE = ("sum", "max")
# src/ir/shapes.js:51-52 (same order)
OPS = ("input", "const") + BINARY + UNARY + ("matmul",) + REDUCE + ("broadcast", "reshape", "transpose")
# Operators of a decoder's training step that the backend has whole kernels for (the reference has none of
# them; its composites would hold the logits, or pass over the values several times).
TRAINING_OPS = ("linearNll", "linearNllGrad", "headNormRope", "headNormRopeGrad", "orthogonalize")
OPS += TRAINING_OPS
MAX_CLASSES = 1 << 24    # class indices and positions are whole numbers in float32
MAX_HEAD = 512
# Of an operand of theirs: the kernels count rows and columns in 31 bits, both hosts bytes in 63.
MAX_DIM, MAX_VALUES = 1 << 30, 1 << 40


class ShapeError(ValueError):
    """A shape rule was broken (src/ir/shapes.js:3-5)."""


def size(shape):
    n = 1
    for d in shape:
        n *= d
    return n


def same_shape(a, b):
    return len(a) == len(b) and all(x == y for x, y in zip(a, b))


def fmt(shape):
    return "[" + ",".join(str(d) for d in shape) + "]"


def _is_int(v):
    return isinstance(v, int) and not isinstance(v, bool)


def check_shape(shape, what):
    if not isinstance(shape, (list, tuple)) or not all(_is_int(d) and d >= 1 for d in shape):
        raise ShapeError(f"{what}: shape must be a list of positive integers, got {shape!r}")


def norm_axis(axis, rank, op):
    """src/ir/shapes.js:17-24."""
    a = axis + rank if axis < 0 else axis
    if not _is_int(a) or a < 0 or a >= rank:
        raise ShapeError(f"{op}: axis {axis} out of range for rank {rank}")
    return a


def broadcast_shapes(a, b):
    """NumPy broadcasting of two shapes, or None (src/ir/shapes.js:27-37)."""
    rank = max(len(a), len(b))
    out = []
    for i in range(rank):
        ia = len(a) - rank + i
        ib = len(b) - rank + i
        da = a[ia] if ia >= 0 else 1
        db = b[ib] if ib >= 0 else 1
        if da != db and da != 1 and db != 1:
            return None
        out.append(max(da, db))
    return out


def broadcasts_to(frm, to):
    """src/ir/shapes.js:40-44."""
    if len(frm) > len(to):
        return False
    lead = len(to) - len(frm)
    return all(d == 1 or d == to[lead + i] for i, d in enumerate(frm))


def infer_shape(op, shapes, attrs):
    """The result shape of ``op`` (src/ir/shapes.js:55-114)."""
    if op not in OPS:
        raise ShapeError(f"unknown op '{op}'")
    if op in TRAINING_OPS:
        return _infer_training(op, shapes, attrs)
    want = {"input": 0, "const": 0, "matmul": 2}.get(op, 2 if op in BINARY else 1)
    if len(shapes) != want:
        raise ShapeError(f"{op}: takes {want} inputs, got {len(shapes)}")
    if op in ("input", "const"):
        check_shape(attrs.get("shape"), op)
        if op == "const":
            v = attrs.get("value")
            ok = isinstance(v, (int, float)) and not isinstance(v, bool) or (
                isinstance(v, (list, tuple)) and len(v) == size(attrs["shape"]))
            if not ok:
                raise ShapeError(f"const: value must be a number or {size(attrs['shape'])} numbers")
        return list(attrs["shape"])
    if op in BINARY:
        if not same_shape(shapes[0], shapes[1]):
            raise ShapeError(f"{op}: shapes {fmt(shapes[0])} and {fmt(shapes[1])} differ; broadcast explicitly")
        return list(shapes[0])
    if op in UNARY:
        return list(shapes[0])
    if op == "matmul":
        a, b = shapes
        if len(a) < 2 or len(b) < 2:
            raise ShapeError(f"matmul: needs rank >= 2, got {fmt(a)} and {fmt(b)}")
        if len(a) != len(b) or not same_shape(a[:-2], b[:-2]):
            raise ShapeError(f"matmul: batch dims of {fmt(a)} and {fmt(b)} differ")
        if a[-1] != b[-2]:
            raise ShapeError(f"matmul: inner dims of {fmt(a)} and {fmt(b)} differ")
        return list(a[:-1]) + [b[-1]]
    if op in REDUCE:
        x = shapes[0]
        axis = norm_axis(attrs["axis"], len(x), op)
        if attrs["axis"] != axis:
            raise ShapeError(f"{op}: axis must be stored normalised")
        if attrs.get("keepDims"):
            return [1 if i == axis else d for i, d in enumerate(x)]
        return [d for i, d in enumerate(x) if i != axis]
    if op == "broadcast":
        check_shape(attrs.get("shape"), op)
        if not broadcasts_to(shapes[0], attrs["shape"]):
            raise ShapeError(f"broadcast: {fmt(shapes[0])} does not broadcast to {fmt(attrs['shape'])}")
        return list(attrs["shape"])
    if op == "reshape":
        check_shape(attrs.get("shape"), op)
        if size(attrs["shape"]) != size(shapes[0]):
            raise ShapeError(f"reshape: {fmt(shapes[0])} has {size(shapes[0])} elements, "
                             f"{fmt(attrs['shape'])} has {size(attrs['shape'])}")
        return list(attrs["shape"])
    if op == "transpose":
        x = shapes[0]
        p = attrs.get("perm")
        ok = isinstance(p, (list, tuple)) and len(p) == len(x) and sorted(p) == list(range(len(x)))
        if not ok:
            raise ShapeError(f"transpose: {p!r} is not a permutation of rank {len(x)}")
        return [x[i] for i in p]
    raise ShapeError(f"no shape rule for '{op}'")


def _number(v):
    if not isinstance(v, (int, float)) or isinstance(v, bool):
        return False
    try:
        return math.isfinite(float(v))
    except OverflowError:   # an int beyond every float
        return False


def _check_eps(op, eps):
    """eps as the kernel takes it, a float32: one above 0 must stay so, or a zero norm is divided by zero."""
    if not _number(eps) or eps < 0 or not math.isfinite(f32(eps)) or (eps > 0 and f32(eps) == 0):
        raise ShapeError(f"{op}: eps must be 0 or a positive float32, got {eps!r}")


def linear_nll_saved(R, d, V):
    """The value linearNll saves for its backward: byte offsets of its parts (the scales at 0, the scaled bias
    at 256; "lse": each row's largest logit and 1 over its sum of exponentials below it) and its size in floats.
    h and W are held as fp16 pairs in blocks of 256 columns."""
    def up(n, k):
        return -(-n // k) * k

    def blocked(n):
        return up(n, 32) if n <= 256 else up(n, 256)
    lse = up(256 + 4 * up(V, 256), 256)
    h = up(lse + 8 * R, 256)
    w = up(h + 4 * R * blocked(d), 256)
    return {"lse": lse, "h": h, "w": w}, up(w + 4 * d * blocked(V), 256) // 4


def _infer_nll(op, shapes, attrs):
    bias = attrs.get("bias")
    if not isinstance(bias, bool):
        raise ShapeError(f"{op}: bias must be true or false")
    if op == "linearNllGrad":   # of the targets, the saved value, the loss's cotangent
        if len(shapes) != 3:
            raise ShapeError(f"{op}: takes 3 inputs, got {len(shapes)}")
        d, V, wrt = attrs.get("d"), attrs.get("V"), attrs.get("wrt")
        if not _is_int(d) or not _is_int(V) or not 1 <= d <= MAX_DIM or not 1 <= V <= MAX_CLASSES:
            raise ShapeError(f"{op}: d and V must be the weight's sizes, got {d!r} and {V!r}")
        t, saved, gy = shapes
        if len(t) != 1 or list(gy) != list(t) or list(saved) != [linear_nll_saved(t[0], d, V)[1]]:
            raise ShapeError(f"{op}: targets {fmt(t)}, saved value {fmt(saved)} and cotangent {fmt(gy)} do not belong "
                             f"to a weight [{d},{V}]")
        if wrt not in ("h", "w", "b") or (wrt == "b" and not bias):
            raise ShapeError(f"{op}: no gradient with respect to {wrt!r}")
        return [t[0], d] if wrt == "h" else [d, V] if wrt == "w" else [V]
    if len(shapes) != 3 + bias:
        raise ShapeError(f"{op}: takes {3 + bias} inputs, got {len(shapes)}")
    h, w = shapes[0], shapes[1]
    if len(h) != 2 or len(w) != 2 or h[1] != w[0]:
        raise ShapeError(f"{op}: rows {fmt(h)} and weight {fmt(w)} must be [R,d] and [d,V]")
    if w[1] > MAX_CLASSES:
        raise ShapeError(f"{op}: {w[1]} classes, at most {MAX_CLASSES} (a class index is a float32)")
    if bias and list(shapes[2]) != [w[1]]:
        raise ShapeError(f"{op}: bias {fmt(shapes[2])} for {w[1]} classes")
    if list(shapes[-1]) != [h[0]]:
        raise ShapeError(f"{op}: targets {fmt(shapes[-1])} for {h[0]} rows")
    out = attrs.get("out")
    if out not in ("loss", "saved"):
        raise ShapeError(f"{op}: out must be 'loss' or 'saved', got {out!r}")
    return [h[0]] if out == "loss" else [linear_nll_saved(h[0], w[0], w[1])[1]]


def _infer_head(op, shapes, attrs):
    back = op == "headNormRopeGrad"
    want = 3 + back
    if len(shapes) != want:
        raise ShapeError(f"{op}: takes {want} inputs, got {len(shapes)}")
    x, gain, pos = shapes[:3]
    if len(x) != 4:
        raise ShapeError(f"{op}: x must be [B,T,H,D], got {fmt(x)}")
    B, T, H, D = x
    if D > MAX_HEAD:
        raise ShapeError(f"{op}: a head of {D} values, at most {MAX_HEAD}")
    if list(gain) != [D]:
        raise ShapeError(f"{op}: gain {fmt(gain)} for heads of {D}")
    if list(pos) not in ([T], [B, T]):
        raise ShapeError(f"{op}: positions {fmt(pos)} must be {fmt([T])} or {fmt([B, T])}")
    r = attrs.get("rotary")
    if not _is_int(r) or r < 0 or r > D or r % 2:
        raise ShapeError(f"{op}: rotary must be an even number of a head's {D} values, got {r!r}")
    for name in ("interleaved", "headsFirst"):
        if not isinstance(attrs.get(name), bool):
            raise ShapeError(f"{op}: {name} must be true or false")
    _check_eps(op, attrs.get("eps"))
    if not _number(attrs.get("base")) or attrs["base"] <= 0:
        raise ShapeError(f"{op}: base must be a number above 0")
    out = [B, H, T, D] if attrs["headsFirst"] else [B, T, H, D]
    if not back:
        return out
    if list(shapes[3]) != out:
        raise ShapeError(f"{op}: cotangent {fmt(shapes[3])} of a value {fmt(out)}")
    wrt = attrs.get("wrt")
    if wrt not in ("x", "gain"):
        raise ShapeError(f"{op}: no gradient with respect to {wrt!r}")
    return list(x) if wrt == "x" else [D]


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)   # the Muon optimiser's quintic
F16_ROOM = 60000.0    # largest scaled value held in fp16, a little below its limit


def newton_schulz_scales(steps, coeffs):
    """Exponents (x, s, p) of the powers of two that scale X, S and P of every Newton-Schulz step into fp16.

    Singular values start in [0, 1] (the Frobenius norm is divided out) and every step maps them by
    a t + b t^3 + c t^5, so the largest singular value after each step, and with it the largest entry that
    X, S = X X^T and P = b S + c S S can have, follow from the extrema of polynomials.  1 % is left for the
    rounding of the products."""
    a, b, c = coeffs
    top, mx, ms, mp = 1.0, 0.0, 0.0, 0.0
    for _ in range(steps):
        s = top * top
        mx, ms = max(mx, top), max(ms, s)
        mp = max(mp, abs(b * s + c * s * s))
        if c != 0 and 0 < -b / (2 * c) < s:
            mp = max(mp, abs(b * b / (4 * c)))
        nxt = abs(a * top + b * top * s + c * top * s * s)
        if c != 0:
            disc = 9 * b * b - 20 * a * c
            roots = [(-3 * b + math.sqrt(disc)) / (10 * c), (-3 * b - math.sqrt(disc)) / (10 * c)] if disc >= 0 else []
        else:
            roots = [-a / (3 * b)] if b != 0 else []
        for t in roots:
            if 0 < t < s:
                q = math.sqrt(t)
                nxt = max(nxt, abs(a * q + b * q * t + c * q * t * t))
        top = nxt * 1.01
    out = []
    for bound in (mx, ms, mp):
        k = 0
        while k < 15 and bound * 1.01 * (2 << k) <= F16_ROOM:
            k += 1
        if not bound * 1.01 * (1 << k) <= F16_ROOM:
            raise ShapeError(f"orthogonalize: coefficients {tuple(coeffs)} let the values grow beyond fp16 in {steps} steps")
        out.append(k)
    return tuple(out)


def _infer_orthogonalize(op, shapes, attrs):
    if len(shapes) != 1:
        raise ShapeError(f"{op}: takes 1 input, got {len(shapes)}")
    x = shapes[0]
    if len(x) < 2:
        raise ShapeError(f"{op}: needs rank >= 2, got {fmt(x)}")
    if size(x[:-2]) > 65535:
        raise ShapeError(f"{op}: {size(x[:-2])} matrices in {fmt(x)}, at most 65535")
    steps, co, eps = attrs.get("steps"), attrs.get("coeffs"), attrs.get("eps")
    if not _is_int(steps) or not 1 <= steps <= 32:
        raise ShapeError(f"{op}: steps must be 1 to 32, got {steps!r}")
    if not isinstance(co, (list, tuple)) or len(co) != 3 or not all(_number(v) and math.isfinite(f32(v)) for v in co):
        raise ShapeError(f"{op}: coeffs must be three float32 numbers, got {co!r}")
    _check_eps(op, eps)
    newton_schulz_scales(steps, co)
    return list(x)


def _infer_training(op, shapes, attrs):
    for s in shapes:
        if any(d > MAX_DIM for d in s) and not (op == "linearNllGrad" and s is shapes[1]) or size(s) > MAX_VALUES:
            raise ShapeError(f"{op}: an operand of shape {fmt(s)}, beyond {MAX_DIM} an axis or {MAX_VALUES} values")
    if op in ("linearNll", "linearNllGrad"):
        return _infer_nll(op, shapes, attrs)
    if op in ("headNormRope", "headNormRopeGrad"):
        return _infer_head(op, shapes, attrs)
    return _infer_orthogonalize(op, shapes, attrs)


class Node:
    __slots__ = ("id", "op", "inputs", "attrs", "shape")

    def __init__(self, id, op, inputs, attrs, shape):
        self.id = id
        self.op = op
        self.inputs = inputs
        self.attrs = attrs
        self.shape = shape

    def __repr__(self):
        return f"Node({self.id}, {self.op}, {self.inputs}, {fmt(self.shape)})"


class Graph:
    """src/ir/graph.js:15-147: raw ``emit`` plus a broadcasting builder."""

    def __init__(self):
        self.nodes = []

    def emit(self, op, inputs=(), attrs=None):
        attrs = {} if attrs is None else attrs
        for i in inputs:
            if not _is_int(i) or i < 0 or i >= len(self.nodes):
                raise ShapeError(f"{op}: input {i} is not a value of this graph")
        shape = infer_shape(op, [self.nodes[i].shape for i in inputs], attrs)
        nid = len(self.nodes)
        self.nodes.append(Node(nid, op, list(inputs), copy.deepcopy(attrs), shape))
        return nid

    def shape(self, nid):
        return self.nodes[nid].shape

    def input_id(self, name):
        for n in self.nodes:
            if n.op == "input" and n.attrs["name"] == name:
                return n.id
        return None

    def inputs(self):
        return [n for n in self.nodes if n.op == "input"]

    def clone(self):
        g = Graph()
        g.nodes = [Node(n.id, n.op, list(n.inputs), copy.deepcopy(n.attrs), list(n.shape)) for n in self.nodes]
        return g

    def to_json(self):
        return {"nodes": [{"op": n.op, "inputs": list(n.inputs), "attrs": copy.deepcopy(n.attrs),
                           "shape": list(n.shape)} for n in self.nodes]}

    @staticmethod
    def from_json(js):
        g = Graph()
        for n in js["nodes"]:
            nid = g.emit(n["op"], n["inputs"], n["attrs"])
            if not same_shape(g.shape(nid), n["shape"]):
                raise ShapeError(f"node {nid}: stored shape {fmt(n['shape'])} but inferred {fmt(g.shape(nid))}")
        return g

    # ---- builder (src/ir/graph.js:66-128) ----
    def input(self, name, shape):
        if self.input_id(name) is not None:
            raise ValueError(f"input '{name}' already exists")
        return self.emit("input", [], {"name": name, "shape": list(shape)})

    def const(self, value, shape=()):
        return self.emit("const", [], {"shape": list(shape), "value": value})

    def broadcast(self, x, shape):
        return x if same_shape(self.shape(x), shape) else self.emit("broadcast", [x], {"shape": list(shape)})

    def _binary(self, op, a, b):
        shape = broadcast_shapes(self.shape(a), self.shape(b))
        if shape is None:
            raise ShapeError(f"{op}: {fmt(self.shape(a))} and {fmt(self.shape(b))} do not broadcast")
        return self.emit(op, [self.broadcast(a, shape), self.broadcast(b, shape)])

    def add(self, a, b): return self._binary("add", a, b)
    def sub(self, a, b): return self._binary("sub", a, b)
    def mul(self, a, b): return self._binary("mul", a, b)
    def div(self, a, b): return self._binary("div", a, b)
    def neg(self, x): return self.emit("neg", [x])
    def exp(self, x): return self.emit("exp", [x])
    def log(self, x): return self.emit("log", [x])
    def relu(self, x): return self.emit("relu", [x])
    def tanh(self, x): return self.emit("tanh", [x])
    def sqrt(self, x): return self.emit("sqrt", [x])
    def step(self, x): return self.emit("step", [x])
    def stop_gradient(self, x): return self.emit("stopGradient", [x])
    def matmul(self, a, b): return self.emit("matmul", [a, b])

    def sum(self, x, axis, keep_dims=False):
        return self.emit("sum", [x], {"axis": norm_axis(axis, len(self.shape(x)), "sum"), "keepDims": keep_dims})

    def max(self, x, axis, keep_dims=False):
        return self.emit("max", [x], {"axis": norm_axis(axis, len(self.shape(x)), "max"), "keepDims": keep_dims})

    def reshape(self, x, shape):
        return x if same_shape(self.shape(x), shape) else self.emit("reshape", [x], {"shape": list(shape)})

    def transpose(self, x, perm=None):
        rank = len(self.shape(x))
        if perm is None:
            perm = list(range(rank))[::-1]
        if all(p == i for i, p in enumerate(perm)):
            return x
        return self.emit("transpose", [x], {"perm": list(perm)})

    def transpose_last2(self, x):
        rank = len(self.shape(x))
        perm = list(range(rank))
        perm[rank - 2], perm[rank - 1] = perm[rank - 1], perm[rank - 2]
        return self.transpose(x, perm)

    # ---- composites (src/ir/graph.js:132-146) ----
    def _shifted(self, x, axis):
        m = self.stop_gradient(self.max(x, axis, True))
        return self.sub(x, m)

    def softmax(self, x, axis=-1):
        z = self.exp(self._shifted(x, axis))
        return self.div(z, self.sum(z, axis, True))

    def log_softmax(self, x, axis=-1):
        z = self._shifted(x, axis)
        return self.sub(z, self.log(self.sum(self.exp(z), axis, True)))

    # ---- operators of a decoder's training step ----
    def linear_nll(self, h, w, bias, targets):
        """-log softmax(h w + bias)[target] of every row, [R]: the cross entropy of a linear head without
        its logits (h [R,d], w [d,V], bias [V] or None, targets [R]: class indices held in float32).

        A row whose target is not in 0 .. V-1 (-1, say, for padding) has loss 0 and no gradient, and
        nothing of its row of h is used.  Gradients: h, w and bias.

        Accurate as float32 in norm: values of h, w and the logits' gradient that are far below the largest of their
        tensor keep an absolute 2^-39 of it (22 bits of their own down to 2^-18 of it)."""
        ins = [h, w] + ([] if bias is None else [bias]) + [targets]
        return self.emit("linearNll", ins, {"bias": bias is not None, "out": "loss"})

    def head_norm_rope(self, x, gain, pos, base=10000.0, eps=1e-6, rotary=None, interleaved=False,
                       heads_first=True):
        """RMS norm over every head of x [B,T,H,D] times gain [D], its first `rotary` values (all of them
        when None) turned by position: pair i by pos * base^(-2i/rotary), pairs being halves apart or, with
        `interleaved`, neighbours.  pos is [T] or [B,T].  The result is [B,H,T,D], what attention reads, or
        x's shape without `heads_first`.  Gradients: x and gain."""
        return self.emit("headNormRope", [x, gain, pos],
                         {"base": base, "eps": eps, "rotary": self.shape(x)[-1] if rotary is None else rotary,
                          "interleaved": interleaved, "headsFirst": heads_first})

    def orthogonalize(self, x, steps=5, coeffs=NEWTON_SCHULZ, eps=1e-7):
        """Newton-Schulz orthogonalisation of the matrix (or every matrix of the stack) x [..., m, n]:
        x / (|x|_F + eps), then `steps` times X = a X + (b S + c S S) X with S = X X^T.  No gradient: it is
        an optimiser's."""
        return self.emit("orthogonalize", [x], {"steps": steps, "coeffs": list(coeffs), "eps": eps})


def strides(shape):
    """Row-major strides (src/interp.js:9-14)."""
    s = [0] * len(shape)
    acc = 1
    for i in range(len(shape) - 1, -1, -1):
        s[i] = acc
        acc *= shape[i]
    return s


def f32(v):
    """Round a Python float to the nearest float32 value (Math.fround)."""
    import struct
    if math.isnan(v):
        return v
    try:
        return struct.unpack("f", struct.pack("f", v))[0]
    except OverflowError:
        return math.copysign(math.inf, v)
