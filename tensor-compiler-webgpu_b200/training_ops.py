"""Launches of the operators of a decoder's training step (ir.TRAINING_OPS).

* ``linearNll`` / ``linearNllGrad``       -- tcb/linear_nll.cuh
* ``headNormRope`` / ``headNormRopeGrad`` -- tcb/head_norm_rope.cuh
* ``orthogonalize``                       -- tcb/orthogonalize.cuh

Each node is one launch of a few kernel calls; the gradients of one node (its ``...Grad`` siblings, which
differ in ``wrt`` only) are one launch with several outputs.  Sizes are run-time parameters, so one module
serves every shape of an operator and only tile widths, a head's layout and Newton-Schulz coefficients are
compiled in.  The library's own lowering (csrc/lower.cpp) makes the same records.
"""
from __future__ import annotations

import math
import struct

from .ir import TRAINING_OPS, newton_schulz_scales, size

SM_COUNT = 148
F16 = 1 << 33          # box_cols flag of a tensor map: 16-bit elements
F16_BM, F16_BK = 128, 32
SCALES_AT, AMAX_AT = 0, 512      # byte offsets in scratch
AMAX_BLOCKS = 2 * SM_COUNT
DZ_BYTES = 256 << 20             # bound of one vocabulary piece's dz


def _up(n, k):
    return -(-n // k) * k


def _f16_stages(bn):
    stage = 2 * F16_BM * F16_BK * 2 + 2 * bn * F16_BK * 2
    return min(8, (227 * 1024 - 2048 - 32768) // stage), stage


def f16_smem(bn):
    """Ring, barriers, staging and 1 KB to align the ring (tcb/gemm_f16x3.cuh)."""
    stages, stage = _f16_stages(bn)
    return stages * stage + 1024 + 32768 + 1024


def f16_bn(M, N, batch=1):
    """Tile width of a split-fp16 product: the widest whose tiles cover the SMs, down to 64."""
    for bn in (256, 128):
        if N > bn // 2 and batch * math.ceil(M / F16_BM) * math.ceil(N / bn) >= SM_COUNT // 2:
            return bn
    return 64


def _symmetric_tiles(n, bn):
    tn = math.ceil(n / bn)
    return sum(tn - i * F16_BM // bn for i in range(math.ceil(n / F16_BM)))


def _operand(off, plane, cols, rows, batch, pitch, mn, bn):
    """The maps of an operand's hi and lo planes: boxes of 64 x F16_BK when its M or N index runs along
    the rows, else of F16_BK x (128 or the tile width)."""
    box = (64 | F16, F16_BK) if mn else (F16_BK | F16, bn)
    return [("scratch", off + p * plane, cols, rows, batch, pitch * 2, rows_stride, *box)
            for p, rows_stride in ((0, rows * pitch * 2), (1, rows * pitch * 2))]


def _gemm(name, M, N, K, batch, bn, maps, params, tiles=None):
    from .codegen import KernelCall
    tiles = batch * math.ceil(M / F16_BM) * math.ceil(N / bn) if tiles is None else tiles
    if tiles >= 1 << 31:
        raise ValueError(f"{name}: {tiles} tiles")
    c = KernelCall(f"{name}_{bn}", (min(SM_COUNT, tiles), 1, 1), (384, 1, 1), f16_smem(bn), [M, N, K, batch, *params])
    c.tma = maps
    return c


def siblings(graph):
    """{node id: [node ids]} of every ...Grad node: the gradients of one node, by operands and attributes."""
    groups, out = {}, {}
    for n in graph.nodes:
        if n.op.endswith("Grad") and n.op in TRAINING_OPS:
            key = (n.op, tuple(n.inputs), repr(sorted((k, v) for k, v in n.attrs.items() if k != "wrt")))
            groups.setdefault(key, []).append(n.id)
            out[n.id] = groups[key]
    return out


# ------------------------------------------------------------------ linearNll
def nll_pieces(R, V):
    """(columns of a piece, pieces): dz of a piece, 4 bytes a value, within DZ_BYTES; whole 256-wide tiles,
    the pieces of about one size."""
    most = max(256, DZ_BYTES // (4 * R) // 256 * 256)
    n = math.ceil(V / most)
    wide = min(_up(math.ceil(V / n), 256), _up(V, 8))
    return wide, math.ceil(V / wide)


def nll_layout(R, d, V, backward):
    dp, vp = _up(d, 8), _up(V, 8)
    bz = f16_bn(R, nll_pieces(R, V)[0] if backward else V)
    at, off = {}, _up(AMAX_AT + 12 * AMAX_BLOCKS, 256) + 256
    at["err"] = off - 256
    piece, _ = nll_pieces(R, V)
    parts = [("h", 4 * R * dp), ("w", 4 * d * vp)]
    if backward:
        parts += [("stat", 16 * R), ("dz", 4 * R * piece), ("db", 4 * math.ceil(R / 32) * V)]
    else:
        parts += [("stat", 4 * R), ("part", 8 * R * math.ceil(V / (bz // 2)))]
    for name, nbytes in parts:
        at[name] = off
        off += _up(nbytes, 256)
    return at, off, bz


def nll_source(bias):
    return f"""// cross entropy of a linear head, {'bias' if bias else 'no bias'}
#include "tcb/common.cuh"
#define TCB_BIAS {int(bias)}
#include "tcb/linear_nll.cuh"
"""


def _nll_prep(R, d, V, at, flags):
    """The scale and split passes both directions begin with."""
    from .codegen import KernelCall
    tail = [R, d, V, at["h"], at["w"], at["stat"], at.get("part", at.get("dz")), at.get("db", 0), 0, flags]
    amax = KernelCall("tcb_nll_amax", (AMAX_BLOCKS, 1, 1), (256, 1, 1), 0, [AMAX_BLOCKS, 0, 0, 0, *tail])
    amax.err_offset = at["err"]
    units = d * math.ceil(V / 1024) + R * math.ceil(d / 1024)
    split = KernelCall("tcb_nll_split", (max(2, min(units, SM_COUNT * 8)), 1, 1), (256, 1, 1), 0,
                       [AMAX_BLOCKS, 0, 0, 0, *tail])
    return [amax, split], tail


def _nll_launch(graph, node):
    from .codegen import KernelCall, Launch
    (R, d), V = graph.nodes[node.inputs[0]].shape, graph.nodes[node.inputs[1]].shape[1]
    dp, vp = _up(d, 8), _up(V, 8)
    at, scratch, bz = nll_layout(R, d, V, False)
    calls, tail = _nll_prep(R, d, V, at, 0)
    maps = (_operand(at["h"], 2 * R * dp, d, R, 1, dp, False, F16_BM) +
            _operand(at["w"], 2 * d * vp, V, d, 1, vp, True, bz))
    gemm = _gemm("tcb_nll_logits", R, V, d, 1, bz, maps, tail)
    gemm.err_offset = at["err"]
    calls.append(gemm)
    calls.append(KernelCall("tcb_nll_finish", (math.ceil(R / 32), 1, 1), (256, 1, 1), 0,
                            [math.ceil(V / (bz // 2)), 0, 0, 0, *tail]))
    return Launch(node.id, node.op, "linear-nll", None, node.inputs, nll_source(node.attrs["bias"]), calls,
                  scratch_bytes=scratch, info={"rnv": (R, d, V), "bn": bz, "path": "tcgen05-f16x3"})


def _nll_grad_launch(graph, ids):
    from .codegen import KernelCall, Launch
    node = graph.nodes[ids[0]]
    (R, d), V = graph.nodes[node.inputs[0]].shape, graph.nodes[node.inputs[1]].shape[1]
    dp, vp = _up(d, 8), _up(V, 8)
    at, scratch, bz = nll_layout(R, d, V, True)
    piece, pieces = nll_pieces(R, V)
    bh, bw = f16_bn(R, d), f16_bn(d, piece)
    want = {graph.nodes[i].attrs["wrt"]: i for i in ids}

    def to(call, wrt):
        if want[wrt] != node.id:
            call.out_node = want[wrt]
        return call
    calls, tail = _nll_prep(R, d, V, at, 1)
    for k in range(pieces):
        v0 = k * piece
        n = min(piece, V - v0)
        zp = _up(n, 8)
        params = tail[:-2] + [v0, 1 | (2 if k else 0)]
        hk = _operand(at["h"], 2 * R * dp, d, R, 1, dp, False, F16_BM)
        hm = _operand(at["h"], 2 * R * dp, d, R, 1, dp, True, F16_BM)
        wk = _operand(at["w"] + 2 * v0, 2 * d * vp, n, d, 1, vp, False, bh)
        wm = _operand(at["w"] + 2 * v0, 2 * d * vp, n, d, 1, vp, True, bz)
        zk = _operand(at["dz"], 2 * R * zp, n, R, 1, zp, False, F16_BM)
        zm = _operand(at["dz"], 2 * R * zp, n, R, 1, zp, True, bw)
        out = [("scratch", at["dz"], n, R, 2, zp * 2, R * zp * 2, 32 | F16, 32)]
        calls.append(_gemm("tcb_nll_dz", R, n, d, 1, bz, hk + wm + out, params))
        if "h" in want:
            calls.append(to(_gemm("tcb_nll_dh", R, d, n, 1, bh, zk + wk, params), "h"))
        if "w" in want:
            calls.append(to(_gemm("tcb_nll_dw", d, n, R, 1, bw, hm + zm, params), "w"))
    for c in calls:
        if c.tma:
            c.err_offset = at["err"]
    if "b" in want:
        calls.append(to(KernelCall("tcb_nll_db", (math.ceil(V / 32), 1, 1), (256, 1, 1), 0, [0, 0, 0, 0, *tail]), "b"))
    return Launch(node.id, node.op, "linear-nll-grad", None, node.inputs, nll_source(node.attrs["bias"]), calls,
                  scratch_bytes=scratch,
                  info={"rnv": (R, d, V), "pieces": pieces, "bn": (bz, bh, bw), "path": "tcgen05-f16x3"})


# ------------------------------------------------------------------ headNormRope
def _head_rows(D, rotary, v):
    """(lanes of a row, rows of a block) with v values a load (tcb/head_norm_rope.cuh, HnRow)."""
    units = math.ceil(rotary / 2 / v) + math.ceil((D - rotary) / (2 * v))
    lanes = 1
    while lanes < min(units, 32):
        lanes *= 2
    return lanes, 256 // lanes


def head_source(D, rotary, interleaved):
    return f"""// head norm and rotation: heads of {D}, {rotary} turned{' in neighbouring pairs' if interleaved else ''}
#include "tcb/common.cuh"
#define TCB_D {D}
#define TCB_ROT {rotary}
#define TCB_INTERLEAVED {int(interleaved)}
#include "tcb/head_norm_rope.cuh"
"""


def _head_launch(graph, ids):
    from .codegen import KernelCall, Launch
    node = graph.nodes[ids[0]]
    B, T, H, D = graph.nodes[node.inputs[0]].shape
    a = node.attrs
    rot = a["rotary"]
    back = node.op == "headNormRopeGrad"
    want = {graph.nodes[i].attrs.get("wrt"): i for i in ids}
    wide = rot % 8 == 0 and D % 4 == 0
    _, rows = _head_rows(D, rot, 4 if wide else 1)
    # a block's rows: `heads` of each of rows / heads tokens.  Few heads at a time let a group keep a
    # token's angles over its other heads; with too few tokens to fill the SMs so, all of them at once
    heads = 1
    while heads * 8 <= H and heads * 2 <= rows:
        heads *= 2
    while heads < H and heads * 2 <= rows and math.ceil(T / (rows // heads)) * B < SM_COUNT * 4:
        heads *= 2
    tiles = math.ceil(T / (rows // heads))
    parts = min(B, max(1, math.ceil(SM_COUNT * 8 / tiles)))
    grid = min(tiles * parts, SM_COUNT * 8)
    flags = (1 if len(graph.nodes[node.inputs[2]].shape) == 1 else 0) | (2 if a["headsFirst"] else 0)
    flags |= (4 if "x" in want else 0) | (8 if "gain" in want else 0)
    eps = struct.unpack("<I", struct.pack("<f", a["eps"]))[0]
    step = struct.unpack("<q", struct.pack("<d", math.log2(a["base"]) / (rot // 2) if rot else 0.0))[0]
    smem = 0
    if "gain" in want:
        smem = 4 * D * max(_head_rows(D, rot, v)[1] for v in ((4, 1) if wide else (1,)))
    main = KernelCall("tcb_head_norm_rope_grad" if back else "tcb_head_norm_rope", (grid, 1, 1), (256, 1, 1), smem,
                      [B, T, H, flags, heads, parts, eps, step])
    calls, scratch = [main], 0
    if back and "x" in want and want["x"] != node.id:
        main.out_node = want["x"]
    if "gain" in want:
        scratch = grid * D * 4
        fin = KernelCall("tcb_head_gain_finish", (math.ceil(D / 32), 1, 1), (1024, 1, 1), 0, [grid])
        if want["gain"] != node.id:
            fin.out_node = want["gain"]
        calls.append(fin)
    return Launch(node.id, node.op, "head-norm-rope-grad" if back else "head-norm-rope", None, node.inputs,
                  head_source(D, rot, a["interleaved"]), calls, scratch_bytes=scratch, info={"bthd": (B, T, H, D), "heads": heads, "parts": parts})


# ------------------------------------------------------------------ orthogonalize
NS_PARTS = 64


def orth_source(steps, coeffs, eps):
    from .codegen import f32_literal
    ex, es, ep = newton_schulz_scales(steps, coeffs)
    return f"""// Newton-Schulz orthogonalisation
#include "tcb/common.cuh"
#define TCB_EX {ex}
#define TCB_ES {es}
#define TCB_EP {ep}
#define TCB_NS_A {f32_literal(coeffs[0])}
#define TCB_NS_B {f32_literal(coeffs[1])}
#define TCB_NS_C {f32_literal(coeffs[2])}
#define TCB_NS_EPS {f32_literal(eps)}
#include "tcb/orthogonalize.cuh"
"""


def _orth_launch(graph, node):
    from .codegen import KernelCall, Launch
    x = graph.nodes[node.inputs[0]].shape
    batch, m, n = size(x[:-2]), x[-2], x[-1]
    a = node.attrs
    tall = m > n
    s = min(m, n)
    xp, sp = _up(n, 8), _up(s, 8)
    xplane, splane = 2 * batch * m * xp, 2 * batch * s * sp
    off = _up(512 + 8 * NS_PARTS * batch, 256) + 256
    err = off - 256
    xs = (off, off + _up(2 * xplane, 256))
    s_at = xs[1] + _up(2 * xplane, 256)
    p_at = s_at + _up(2 * splane, 256)
    scratch = p_at + _up(2 * splane, 256)
    bs, bx = f16_bn(s, s, batch), f16_bn(m, n, batch)
    parts = max(1, min(NS_PARTS, math.ceil(m * n / 4096)))
    norm = KernelCall("tcb_orth_norm", (parts, batch, 1), (256, 1, 1), 0, [parts, 0, 0, 0, m, n])
    norm.err_offset = err
    split = KernelCall("tcb_orth_split", (max(1, min(m * math.ceil(n / 1024), SM_COUNT * 8)), batch, 1), (256, 1, 1), 0,
                       [parts, 0, 0, 0, m, n, xs[0]])
    calls = [norm, split]
    sym = batch * _symmetric_tiles(s, bs)

    def x_map(off, mn, bn):
        return _operand(off, xplane, n, m, batch, xp, mn, bn)

    def s_map(off, bn):
        return _operand(off, splane, s, s, batch, sp, False, bn)

    def out(off, rows, cols, pitch):
        return [("scratch", off, cols, rows, 2 * batch, pitch * 2, rows * pitch * 2, 32 | F16, 32)]
    for k in range(a["steps"]):
        cur, nxt = xs[k % 2], xs[1 - k % 2]
        last = k == a["steps"] - 1
        params = [m, n, cur, nxt, s_at, p_at, int(last)]
        calls.append(_gemm("tcb_orth_gram_tall" if tall else "tcb_orth_gram_wide", s, s, max(m, n), batch, bs,
                           x_map(cur, tall, F16_BM) + x_map(cur, tall, bs) + out(s_at, s, s, sp), params, sym))
        calls.append(_gemm("tcb_orth_poly", s, s, s, batch, bs,
                           s_map(s_at, F16_BM) + s_map(s_at, bs) + out(p_at, s, s, sp), params, sym))
        ab = x_map(cur, False, F16_BM) + s_map(p_at, bx) if tall else s_map(p_at, F16_BM) + x_map(cur, True, bx)
        calls.append(_gemm("tcb_orth_apply_tall" if tall else "tcb_orth_apply_wide", m, n, s, batch, bx, ab + out(nxt, m, n, xp), params))
    for c in calls:
        if c.tma:
            c.err_offset = err
    return Launch(node.id, node.op, "orthogonalize", None, node.inputs,
                  orth_source(a["steps"], a["coeffs"], a["eps"]), calls, scratch_bytes=scratch,
                  info={"mn": (batch, m, n), "bn": (bs, bx), "path": "tcgen05-f16x3"})


def training_launch(graph, node, groups):
    """The launch of a TRAINING_OPS node, or None for a gradient that an earlier sibling's launch computes."""
    ids = groups.get(node.id, [node.id])
    if ids[0] != node.id:
        return None
    if node.op == "linearNll":
        lau = _nll_launch(graph, node)
    elif node.op == "linearNllGrad":
        lau = _nll_grad_launch(graph, ids)
    elif node.op in ("headNormRope", "headNormRopeGrad"):
        lau = _head_launch(graph, ids)
    else:
        lau = _orth_launch(graph, node)
    if len(ids) > 1:
        lau.nodes = list(ids)
    lau.bytes = 4 * (sum(size(graph.nodes[i].shape) for i in dict.fromkeys(lau.inputs)) +
                     sum(size(graph.nodes[i].shape) for i in ids))
    return lau
