"""Launches of the operators of a decoder's training step (ir.TRAINING_OPS).

* ``linearNll`` / ``linearNllGrad``       -- tcb/linear_nll.cuh; a few rows' loss alone tcb/nll_rows.cuh
* ``headNormRope`` / ``headNormRopeGrad`` -- tcb/head_norm_rope.cuh
* ``orthogonalize``                       -- tcb/orthogonalize.cuh, tcb/orth_small.cuh

Each node is one launch of a few kernel calls.  Siblings -- the gradients of one node, which differ in
``wrt`` only; a loss and what it saves for its backward, which differ in ``out`` -- are one launch with several
outputs.  Sizes are run-time parameters, so one module
serves every shape of an operator and only tile widths, a head's layout and Newton-Schulz coefficients are
compiled in.  The library's own lowering (csrc/lower.cpp) makes the same records.
"""
from __future__ import annotations

import math
import struct
from collections import namedtuple

from .ir import TRAINING_OPS, linear_nll_saved, newton_schulz_scales, size

SM_COUNT = 148
F16 = 1 << 33          # box_cols flags of a tensor map: 16-bit elements,
PAIR = 1 << 34         # two planes (hi and lo) a box
F16_BM, F16_BK = 128, 32
F16_EXTRA = 256 + 8 * 128 + 8 * 4096 + 1024   # beside the ring: barriers, vectors, staging, and to align it
AMAX_BLOCKS = 4 * SM_COUNT
DZ_BYTES = 128 << 20             # bound of one vocabulary piece's dz
CTRL_BYTES = 4 * (4 + 8 * 2 * SM_COUNT)   # error word, and a counter per epilogue warp of a divided tile


def _up(n, k):
    return -(-n // k) * k


class Tile(namedtuple("Tile", "bn ctas")):
    """A product's tile: ctas * 128 rows x bn columns.  A pair of SMs loads 128 rows of A and half of B's columns
    each."""
    def __str__(self):
        return f"{self.bn}x2" if self.ctas == 2 else str(self.bn)

    @property
    def cols(self):
        """Columns of B a CTA loads."""
        return self.bn // self.ctas


def _f16_stages(tile):
    stage = 2 * F16_BM * F16_BK * 2 + 2 * tile.cols * F16_BK * 2
    return min(8, (227 * 1024 - F16_EXTRA) // stage), stage


def f16_smem(tile):
    """Bytes of shared memory (tcb/gemm_f16x3.cuh)."""
    stages, stage = _f16_stages(tile)
    return stages * stage + F16_EXTRA


def f16_tiles(M, N, tile, symmetric):
    rows = F16_BM * tile.ctas
    tm, tn = math.ceil(M / rows), math.ceil(N / tile.bn)
    return sum(tn - i * rows // tile.bn for i in range(tm)) if symmetric else tm * tn


# Nanoseconds of a split-fp16 product by tile, as measured in bursts with every SM busy: a K step of 16 of one tile,
# without its epilogue's share; an epilogue; the exchange of a divided tile's partial sums, at all and for each part.
F16_COST = {Tile(256, 2): (275, 6600, 3000, 2500), Tile(128, 2): (173, 3600, 1500, 1600),
            Tile(128, 1): (180, 3000, 1500, 1200), Tile(64, 1): (140, 1500, 1000, 700)}


def f16_plan(M, N, K, batch, chunk, symmetric=False, only=None):
    """(tile, grid, whole tiles, quantum) of a product (tcb/gemm_f16x3.cuh), the cheapest by F16_COST; with
    `only` whole tiles of that kind.

    Tiles go whole to the SMs in waves, or, where they are fewer than the SMs, in pieces of `quantum` chains
    of `chunk` K indices.  Dividing the last wave of more tiles than that does not pay: the CTAs then no
    longer read the same operands at the same time (4096 x 1024 products of K 8192, 128 of 148 SMs, 146 us
    whole, 216 divided)."""
    best = None
    steps = math.ceil(K / 16)
    for tile, (step, epi, once, part) in F16_COST.items():
        bn, ctas = tile
        units = SM_COUNT // ctas
        if tile != only if only else (bn > 64 and N <= bn // 2) or M <= F16_BM * (ctas - 1):
            continue
        tiles = batch * f16_tiles(M, N, tile, symmetric)
        plans = [(math.ceil(tiles / units) * (steps * step + epi), tile, min(units, tiles) * ctas, tiles, 1)]
        for q in (1, 2, 4, 8, 16, 32, 64):
            per = math.ceil(K / (256 * q))
            if only or tiles >= units or per == 1:
                break
            grid = min(units, tiles * per)
            run = math.ceil(tiles * per / grid)
            pieces = per if run == 1 else per // run + 2
            plans.append((run * q * 16 * step + once + pieces * part + epi, tile, grid * ctas, 0, q * (256 // chunk)))
        for p in plans:
            if best is None or p[0] < best[0]:
                best = p
    return best[1:]


def f16_partial_bytes(grid, whole, tiles, tile):
    return 0 if whole == tiles else 2 * grid * F16_BM * tile.bn * 4


def _operand(off, plane, cols, rows, batch, pitch, mn, box_rows, region="scratch"):
    """The map of an operand's hi and lo planes, one behind the other for each matrix: boxes of 64 x F16_BK when
    its M or N index runs along the rows, else of F16_BK x the rows of A or columns of B that a CTA loads."""
    box = (64 | F16 | PAIR, F16_BK) if mn else (F16_BK | F16 | PAIR, box_rows)
    assert plane == batch * rows * pitch * 2
    return [(region, off, cols, rows, 2 * batch, pitch * 2, rows * pitch * 2, *box)]


def _blocked(region, off, rows, cols, pitch, box_cols, box_rows):
    """The map of a matrix stored in blocks of 256 columns (rows of `pitch`), hi and lo planes of a block side
    by side."""
    return [(region, off, pitch, rows, 2 * math.ceil(cols / 256), pitch * 2, rows * pitch * 2, box_cols | F16 | PAIR, box_rows)]


def _pitch(cols):
    return min(256, _up(cols, 32))


def _blocked_operand(region, off, rows, cols, pitch, mn, box_rows):
    return _blocked(region, off, rows, cols, pitch, *((64, F16_BK) if mn else (F16_BK, box_rows)))


def _at(index, off):
    """A tensor map's place in a launch operand, `off` bytes in (region 'in_at')."""
    return off << 3 | index


def _gemm(name, M, N, K, batch, plan, part_at, maps, params, symmetric=False):
    from .codegen import KernelCall
    tile, grid, whole, quantum = plan
    tiles = batch * f16_tiles(M, N, tile, symmetric)
    if tiles >= 1 << 31:
        raise ValueError(f"{name}: {tiles} tiles")
    c = KernelCall(f"{name}_{tile}", (grid, 1, 1), (384, 1, 1), f16_smem(tile),
                   [M | N << 32, K | batch << 32, whole | quantum << 32, part_at, *params])
    c.tma = maps
    return c, f16_partial_bytes(grid, whole, tiles, tile)


def siblings(graph):
    """{node id: [node ids]}: the outputs of one launch, nodes that differ in which output they are only."""
    groups, out = {}, {}
    for n in graph.nodes:
        which = n.attrs.get("wrt", n.attrs.get("out")) if n.op in TRAINING_OPS else None
        if which is None:
            continue
        key = (n.op, tuple(n.inputs), repr(sorted((k, v) for k, v in n.attrs.items() if k not in ("wrt", "out"))))
        for g in groups.setdefault(key, []):
            if which not in g:
                break
        else:
            g = {}
            groups[key].append(g)
        g[which] = n.id
        out[n.id] = g
    return {i: list(g.values()) for i, g in out.items()}


# ------------------------------------------------------------------ linearNll
NLL_CHUNK = 256
# Rows (in 32s) of a forward whose tiles, columns (in 32s) of a backward whose row sums are joined in the
# product's own kernel, and the most parts a warp then adds up on its own
JOIN_COUNTERS, JOIN_PARTS = 512, 4
NLL_CTRL_BYTES = CTRL_BYTES + 4 * JOIN_COUNTERS
NLL_ADD, NLL_JOIN, NLL_NO_LOSS, NLL_DB = 1, 2, 4, 8


def _joined(groups, parts):
    """Joining in the product's kernel saves a launch (64 x 64 x 65: 24.9 us to 22.8), but every part's warp waits for
    its stores and an atomic (4095 x 256 x 8192 with up to 64 parts: 231 us to 269): for few parts only."""
    return groups <= JOIN_COUNTERS and parts <= JOIN_PARTS


def nll_pieces(R, V):
    """(columns of a piece, pieces): dz of a piece, 4 bytes a value, within DZ_BYTES; whole 256-wide tiles,
    the pieces of about one size."""
    most = max(256, DZ_BYTES // (4 * R) // 256 * 256)
    n = math.ceil(V / most)
    wide = min(_up(math.ceil(V / n), 256), _up(V, 32))
    return wide, math.ceil(V / wide)


def nll_source(bias, rows=False):
    return f"""// cross entropy of a linear head, {'bias' if bias else 'no bias'}
#include "tcb/common.cuh"
#define TCB_BIAS {int(bias)}
#include "tcb/{'nll_rows' if rows else 'linear_nll'}.cuh"
"""


# Most rows of a loss without a backward that read W as it is (tcb/nll_rows.cuh) instead of splitting it for the tensor
# core.  16 rows at d x V, us: 64 x 65 12.3 against 12.3, 256 x 8192 14.3 : 25.8, 1024 x 32000 69.8 : 125.9, 1024 x
# 131072 228 : 464; 32 rows at 1024 x 32000 166 : 128, and their sums would take twice the registers.
NLL_ROWS = 16


def _nll_rows_launch(graph, node):
    """A few rows' loss alone (tcb/nll_rows.cuh)."""
    from .codegen import KernelCall, Launch
    (R, d), V = graph.nodes[node.inputs[0]].shape, graph.nodes[node.inputs[1]].shape[1]
    rows = next(k for k in (4, 8, 16) if R <= k)
    blocks = math.ceil(V / 128)
    # parts of d: blocks for every SM four times, at least 64 indices a part
    parts = min(8, max(1, 4 * SM_COUNT // blocks), math.ceil(d / 64))
    per = math.ceil(d / parts)
    parts = math.ceil(d / per)
    at, end = _regions(("sums", 4 * parts * R * V if parts > 1 else 0), ("zt", 4 * R), ("stats", 8 * R * math.ceil(V / 32)))
    params = [parts, per, at["zt"], at["stats"], R, d, V]
    calls = [KernelCall(f"tcb_nll_rows_{rows}", (blocks, parts, 1), (256, 1, 1), 0, params)]
    if parts > 1:
        calls.append(KernelCall("tcb_nll_rows_add", (math.ceil(V / 256), R, 1), (256, 1, 1), 0, params))
    calls.append(KernelCall("tcb_nll_rows_finish", (R, 1, 1), (1024, 1, 1), 0, params))
    return Launch(node.id, node.op, "linear-nll", None, node.inputs, nll_source(node.attrs["bias"], rows=True), calls,
                  scratch_bytes=end, info={"rnv": (R, d, V), "parts": parts, "path": "fma"})


def _regions(*parts):
    """{name: byte offset} of scratch regions one behind the other, and their end."""
    at, off = {}, 0
    for name, nbytes in parts:
        at[name] = off
        off += _up(nbytes, 256)
    return at, off


def _nll_launch(graph, ids):
    from .codegen import KernelCall, Launch
    by = {graph.nodes[i].attrs["out"]: i for i in ids}
    node = graph.nodes[ids[0]]
    (R, d), V = graph.nodes[node.inputs[0]].shape, graph.nodes[node.inputs[1]].shape[1]
    if "saved" not in by and R <= NLL_ROWS:
        return _nll_rows_launch(graph, node)
    inner, floats = linear_nll_saved(R, d, V)
    plan = f16_plan(R, V, d, 1, NLL_CHUNK)
    tile = plan[0]
    halves = math.ceil(V / (tile.bn // 2))
    at, end = _regions(("amax", 8 * AMAX_BLOCKS), ("err", NLL_CTRL_BYTES), ("zt", 4 * R), ("part", 8 * R * halves),
                       ("loss", 0 if "loss" in by else 4 * R), ("saved", 0 if "saved" in by else 4 * floats))
    joined = _joined(math.ceil(R / 32), halves)
    flags = (NLL_JOIN if joined else 0) | (0 if "loss" in by else NLL_NO_LOSS)
    tail = [R, d, V, at["saved"], inner["lse"], inner["h"], inner["w"], at["zt"], at["part"], flags]
    if "saved" in by:
        def saved(off):
            return "out", off
    else:
        def saved(off):
            return "scratch", at["saved"] + off
    maps = (_blocked_operand(*saved(inner["h"]), R, d, _pitch(d), False, F16_BM) +
            _blocked_operand(*saved(inner["w"]), d, V, _pitch(V), True, tile.cols))
    blocks = max(1, min(AMAX_BLOCKS, math.ceil((R * d + d * V) / 2048)))
    units = d * math.ceil(V / 1024) + R * math.ceil(d / 1024)
    gemm, partial = _gemm("tcb_nll_logits", R, V, d, 1, plan, end, maps, tail)
    calls = [KernelCall("tcb_nll_amax", (blocks, 1, 1), (256, 1, 1), 0, [blocks, 0, 0, 0, *tail]),
             KernelCall("tcb_nll_split", (max(2, min(units, SM_COUNT * 8)), 1, 1), (256, 1, 1), 0, [blocks, 0, 0, 0, *tail]),
             gemm]
    if not joined:
        calls.append(KernelCall("tcb_nll_finish", (math.ceil(R / 32), 1, 1), (256, 1, 1), 0, [halves, 0, 0, 0, *tail]))
    calls[0].err_offset = gemm.err_offset = at["err"]
    if "saved" in by:   # `out` is then the saved value, which the product's maps lie in, and the loss an address
        for c in calls:
            c.ptr_params = ((14, by["saved"]),) + (((7, by["loss"]),) if "loss" in by else ())
            if by["saved"] != node.id:
                c.out_node = by["saved"]
    return Launch(node.id, node.op, "linear-nll", None, node.inputs, nll_source(node.attrs["bias"]), calls,
                  scratch_bytes=end + _up(partial, 256),
                  info={"rnv": (R, d, V), "tile": str(tile), "ctrl_bytes": _up(NLL_CTRL_BYTES, 64), "path": "tcgen05-f16x3"})


def _nll_grad_launch(graph, ids):
    from .codegen import KernelCall, Launch
    node = graph.nodes[ids[0]]
    R, (d, V) = graph.nodes[node.inputs[0]].shape[0], (node.attrs["d"], node.attrs["V"])
    inner, _ = linear_nll_saved(R, d, V)
    piece, pieces = nll_pieces(R, V)
    want = {graph.nodes[i].attrs["wrt"]: i for i in ids}
    at, end = _regions(("scale", 256), ("err", NLL_CTRL_BYTES), ("dz", 4 * R * _up(piece, 256 if piece > 256 else 32)),
                       ("db", 4 * math.ceil(R / 32) * V if "b" in want else 0))
    tail = [R, d, V, 0, inner["lse"], inner["h"], inner["w"], at["db"]]
    joined = "b" in want and _joined(math.ceil(V / 32), math.ceil(R / 32))
    calls, partial = [], 0

    # A piece's logits are the forward's, bit for bit: by its own plan where the piece is all of the vocabulary, else
    # by its tile (several pieces have more tiles than there are SMs: neither divides them).  Computed in another
    # order they would be off by roundings of the logits' size, and a row's largest no longer the one subtracted.
    forward = f16_plan(R, V, d, 1, NLL_CHUNK)

    def add(name, wrt, M, N, K, maps, params, plan=None):
        nonlocal partial
        plan = plan or f16_plan(M, N, K, 1, NLL_CHUNK)
        c, nbytes = _gemm(name, M, N, K, 1, plan, end, maps(plan[0].cols), params)
        c.err_offset = at["err"]
        if wrt is not None and want[wrt] != node.id:
            c.out_node = want[wrt]
        partial = max(partial, nbytes)
        calls.append(c)
    for k in range(pieces):
        v0 = k * piece
        n = min(piece, V - v0)
        params = [*tail, v0, (NLL_ADD if k else 0) | (NLL_JOIN if joined else 0) | (NLL_DB if "b" in want else 0)]
        w_at = inner["w"] + (4 * d * v0 if v0 else 0)   # pieces begin with a block

        def h(mn):
            return _blocked_operand("in_at", _at(1, inner["h"]), R, d, _pitch(d), mn, F16_BM)

        def w(mn, box_rows):
            return _blocked_operand("in_at", _at(1, w_at), d, n, _pitch(V), mn, box_rows)

        def z(mn, box_rows):
            return _blocked_operand("scratch", at["dz"], R, n, _pitch(n), mn, box_rows)
        out = _blocked("scratch", at["dz"], R, n, _pitch(n), 32, 32)
        add("tcb_nll_dz", None, R, n, d, lambda cols: h(False) + w(True, cols) + out, params,
            forward if pieces == 1 else f16_plan(R, n, d, 1, NLL_CHUNK, only=forward[0]))
        if joined:
            calls[-1].ptr_params = ((14, want["b"]),)
        ph, pw = f16_plan(R, d, n, 1, NLL_CHUNK), f16_plan(d, n, R, 1, NLL_CHUNK)
        if "h" in want and "w" in want and ph[0].ctas == pw[0].ctas == 1 and ph[1] + pw[1] <= SM_COUNT:
            # both find room side by side
            c, hb = _gemm("tcb_nll_both", R, d, n, 1, ph, end, z(False, F16_BM) + w(False, ph[0].cols) + h(True) + z(True, pw[0].cols), params)
            wb = f16_partial_bytes(pw[1], pw[2], f16_tiles(d, n, pw[0], False), pw[0])
            c.name = f"tcb_nll_both_{ph[0]}_{pw[0]}"
            c.grid, c.smem = (ph[1] + pw[1], 1, 1), max(f16_smem(ph[0]), f16_smem(pw[0]))
            c.params[7:9] = [pw[2] | pw[3] << 32, end + _up(hb, 256)]
            c.params += [ph[1]]
            c.ptr_params = ((9, want["w"]),)
            c.err_offset = at["err"]
            if want["h"] != node.id:
                c.out_node = want["h"]
            partial = max(partial, _up(hb, 256) + wb)
            calls.append(c)
            continue
        if "h" in want:
            add("tcb_nll_dh", "h", R, d, n, lambda cols: z(False, F16_BM) + w(False, cols), params)
        if "w" in want:
            add("tcb_nll_dw", "w", d, n, R, lambda cols: h(True) + z(True, cols), params)
    if "b" in want and not joined:
        db = KernelCall("tcb_nll_db", (math.ceil(V / 32), 1, 1), (256, 1, 1), 0, [0, 0, 0, 0, *tail, 0, 0])
        if want["b"] != node.id:
            db.out_node = want["b"]
        calls.append(db)
    # no pass of its own comes first to clear the control block of a one-off run
    clear = KernelCall("tcb_gemm_prep", (1, 1, 1), (128, 1, 1))
    clear.err_offset = at["err"]
    return Launch(node.id, node.op, "linear-nll-grad", None, node.inputs, nll_source(node.attrs["bias"]), [clear] + calls,
                  scratch_bytes=end + _up(partial, 256),
                  info={"rnv": (R, d, V), "pieces": pieces, "ctrl_bytes": _up(NLL_CTRL_BYTES, 64), "path": "tcgen05-f16x3"})


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
    steps = math.ceil(T / (rows // heads)) * B * math.ceil(H / heads)
    grid = min(steps, SM_COUNT * (2 if back else 4))   # one wave of as many CTAs as the kernel's registers allow
    flags = (1 if len(graph.nodes[node.inputs[2]].shape) == 1 else 0) | (2 if a["headsFirst"] else 0)
    flags |= (4 if "x" in want else 0) | (8 if "gain" in want else 0)
    eps = struct.unpack("<I", struct.pack("<f", a["eps"]))[0]
    step = struct.unpack("<q", struct.pack("<d", math.log2(a["base"]) / (rot // 2) if rot else 0.0))[0]
    smem = 0
    if "gain" in want:
        smem = 4 * D * max(_head_rows(D, rot, v)[1] for v in ((4, 1) if wide else (1,)))
    main = KernelCall("tcb_head_norm_rope_grad" if back else "tcb_head_norm_rope", (grid, 1, 1), (256, 1, 1), smem,
                      [B, T, H, flags, heads, eps, step])
    calls, scratch = [main], 0
    if back and "x" in want and want["x"] != node.id:
        main.out_node = want["x"]
    if "gain" in want:
        scratch = grid * D * 4
        fin = KernelCall("tcb_head_gain_finish", (math.ceil(D / 8), 1, 1), (1024, 1, 1), 0, [grid])
        if want["gain"] != node.id:
            fin.out_node = want["gain"]
        calls.append(fin)
    return Launch(node.id, node.op, "head-norm-rope-grad" if back else "head-norm-rope", None, node.inputs,
                  head_source(D, rot, a["interleaved"]), calls, scratch_bytes=scratch, info={"bthd": (B, T, H, D), "heads": heads})


# ------------------------------------------------------------------ orthogonalize
NS_PARTS = 512
NS_CHUNK = 128


ORTH_SMALL = ((64, 512), (128, 128))   # (short, long) sides of matrices that fit one SM


def orth_small(s, long):
    """The (short, long) limits of the one-SM form a matrix fits, or None."""
    for rows, cols in ORTH_SMALL:
        if s <= rows and long <= cols:
            return rows, cols
    return None


def orth_source(steps, coeffs, eps, small=None):
    from .codegen import f32_literal
    ex, es, ep = newton_schulz_scales(steps, coeffs)
    limits = f"#define TCB_ROWS {small[0]}\n#define TCB_COLS {small[1]}\n" if small else ""
    return f"""// Newton-Schulz orthogonalisation{' on one SM' if small else ''}
#include "tcb/common.cuh"
{limits}#define TCB_EX {ex}
#define TCB_ES {es}
#define TCB_EP {ep}
#define TCB_NS_A {f32_literal(coeffs[0])}
#define TCB_NS_B {f32_literal(coeffs[1])}
#define TCB_NS_C {f32_literal(coeffs[2])}
#define TCB_NS_EPS {f32_literal(eps)}
#include "tcb/{'orth_small' if small else 'orthogonalize'}.cuh"
"""


def _orth_launch(graph, node):
    from .codegen import KernelCall, Launch
    x = graph.nodes[node.inputs[0]].shape
    batch, m, n = size(x[:-2]), x[-2], x[-1]
    a = node.attrs
    tall = m > n
    s = min(m, n)
    small = orth_small(s, max(m, n))
    if small:
        rows, cols = small
        block = 2 * rows * 128
        c = KernelCall("tcb_orth_small", (batch, 1, 1), (256, 1, 1), (cols // 64 + 2 * (rows // 64)) * block + 16384 + 1024,
                       [m, n, a["steps"]])
        c.err_offset = 0
        return Launch(node.id, node.op, "orthogonalize", None, node.inputs, orth_source(a["steps"], a["coeffs"], a["eps"], small),
                      [c], scratch_bytes=256, info={"mn": (batch, m, n), "ctrl_bytes": 64, "path": "tcgen05-f16x3"})
    xp, sp = _up(n, 8), _up(s, 8)
    xplane, splane = 2 * batch * m * xp, 2 * batch * s * sp
    parts = max(1, min(NS_PARTS, math.ceil(m * n / 4096)))
    at, end = _regions(("parts", 8 * parts * batch), ("err", CTRL_BYTES), ("x0", 2 * xplane), ("x1", 2 * xplane),
                       ("s", 2 * splane), ("p", 2 * splane))
    gram, poly = f16_plan(s, s, max(m, n), batch, NS_CHUNK, True), f16_plan(s, s, s, batch, NS_CHUNK, True)
    app = f16_plan(m, n, s, batch, NS_CHUNK)
    norm = KernelCall("tcb_orth_norm", (parts, batch, 1), (256, 1, 1), 0, [parts, 0, 0, 0, m, n])
    norm.err_offset = at["err"]
    split = KernelCall("tcb_orth_split", (max(1, min(m * math.ceil(n / 1024), SM_COUNT * 8)), batch, 1), (256, 1, 1), 0,
                       [parts, 0, 0, 0, m, n, at["x0"]])
    calls, partial = [norm, split], 0

    def x_map(off, mn, box_rows):
        return _operand(off, xplane, n, m, batch, xp, mn, box_rows)

    def s_map(off, box_rows):
        return _operand(off, splane, s, s, batch, sp, False, box_rows)

    def out(off, rows, cols, pitch):
        return [("scratch", off, cols, rows, 2 * batch, pitch * 2, rows * pitch * 2, 32 | F16 | PAIR, 32)]
    for k in range(a["steps"]):
        cur, nxt = (at["x0"], at["x1"]) if k % 2 == 0 else (at["x1"], at["x0"])
        params = [m, n, cur, nxt, at["s"], at["p"], int(k == a["steps"] - 1)]
        ab = x_map(cur, False, F16_BM) + s_map(at["p"], app[0].cols) if tall else s_map(at["p"], F16_BM) + x_map(cur, True, app[0].cols)
        for c, nbytes in (
                _gemm("tcb_orth_gram_tall" if tall else "tcb_orth_gram_wide", s, s, max(m, n), batch, gram, end,
                      x_map(cur, tall, F16_BM) + x_map(cur, tall, gram[0].cols) + out(at["s"], s, s, sp), params, True),
                _gemm("tcb_orth_poly", s, s, s, batch, poly, end,
                      s_map(at["s"], F16_BM) + s_map(at["s"], poly[0].cols) + out(at["p"], s, s, sp), params, True),
                _gemm("tcb_orth_apply_tall" if tall else "tcb_orth_apply_wide", m, n, s, batch, app, end,
                      ab + out(nxt, m, n, xp), params)):
            c.err_offset = at["err"]
            calls.append(c)
            partial = max(partial, nbytes)
    return Launch(node.id, node.op, "orthogonalize", None, node.inputs,
                  orth_source(a["steps"], a["coeffs"], a["eps"]), calls, scratch_bytes=end + _up(partial, 256),
                  info={"mn": (batch, m, n), "tiles": (str(gram[0]), str(poly[0]), str(app[0])), "ctrl_bytes": _up(CTRL_BYTES, 64), "path": "tcgen05-f16x3"})


def training_launch(graph, node, groups):
    """The launch of a TRAINING_OPS node, or None for one that an earlier sibling's launch computes."""
    ids = groups.get(node.id, [node.id])
    if ids[0] != node.id:
        return None
    if node.op == "linearNll":
        lau = _nll_launch(graph, ids)
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
