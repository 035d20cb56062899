"""The workloads of the framework's training operators, in plain torch and through the graph compiler.

Three operators of a decoder's training step:

* ``nll``  -- softmax cross entropy of a linear head over a vocabulary (``Graph.linear_nll``), alone
  (evaluation) or with the gradients of the rows, the head's weight and its bias (training);
* ``head`` -- RMS norm of every query / key head, rotation by position and the move of the head axis in
  front of the tokens (``Graph.head_norm_rope``), alone or with the gradients of the input and the gain;
* ``orth`` -- Newton-Schulz orthogonalisation of a matrix (``Graph.orthogonalize``), or of a stack of them.

Every value is float32, as in the framework's graphs; token indices and positions are whole numbers held
in float32.  With ``own`` false ``run`` computes the plain form, with ``own`` true it replays the resident
program that a user's step keeps.
"""
import importlib
import math

import torch

own = False

PKG = "tensor-compiler-webgpu_b200"
NS = (3.4445, -4.7750, 2.0315)     # Newton-Schulz coefficients of the Muon optimiser
EPS_ROOT = 1e-6                    # RMS norm
EPS_NORM = 1e-7                    # Frobenius norm


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the character model's head (V = 65) on one sequence of 64 tokens: a step of launches only
        {"name": "nll-train-64x64x65", "op": "nll", "R": 64, "d": 64, "V": 65, "train": True, "skip": 0.0},
        # a small model's head on 4095 tokens, a tenth of them padding that takes no loss
        {"name": "nll-train-4095x256x8192", "op": "nll", "R": 4095, "d": 256, "V": 8192, "train": True, "skip": 0.1},
        # a training step's head at full width, the vocabulary of odd size
        {"name": "nll-train-8192x1024x50001", "op": "nll", "R": 8192, "d": 1024, "V": 50001, "train": True, "skip": 0.0},
        # scoring held-out text with a large vocabulary: forward only
        {"name": "nll-eval-16384x1024x131072", "op": "nll", "R": 16384, "d": 1024, "V": 131072, "train": False,
         "skip": 0.0},
        # one new token's queries: a call that is all latency
        {"name": "head-1x1x4x64", "op": "head", "B": 1, "T": 1, "H": 4, "D": 64, "rotary": 64, "interleaved": False,
         "shared": True, "start": 255, "train": False},
        # odd counts: 3 packed sequences with positions of their own, half of an 80-wide head rotated in pairs
        {"name": "head-train-3x1001x5x80", "op": "head", "B": 3, "T": 1001, "H": 5, "D": 80, "rotary": 40,
         "interleaved": True, "shared": False, "start": 0, "train": True},
        # the queries of one block of the benchmark's transformer (batch 512, 256 tokens, 4 heads of 64)
        {"name": "head-train-512x256x4x64", "op": "head", "B": 512, "T": 256, "H": 4, "D": 64, "rotary": 64,
         "interleaved": False, "shared": True, "start": 0, "train": True},
        # long sequences far from the start, 32 heads of 128
        {"name": "head-train-2x8191x32x128", "op": "head", "B": 2, "T": 8191, "H": 32, "D": 128, "rotary": 128,
         "interleaved": False, "shared": True, "start": 1000000, "train": True},
        # a weight of the reference's 64-wide transformer
        {"name": "orth-64x64", "op": "orth", "B": 1, "m": 64, "n": 64},
        # the four blocks' MLP weights of the benchmark's transformer as one stack
        {"name": "orth-4x256x1024", "op": "orth", "B": 4, "m": 256, "n": 1024},
        # an odd tall weight
        {"name": "orth-4095x1000", "op": "orth", "B": 1, "m": 4095, "n": 1000},
        # a large square weight
        {"name": "orth-4096x4096", "op": "orth", "B": 1, "m": 4096, "n": 4096},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("nll", "head", "orth"))
    if op == "nll":
        while True:
            c = {"op": op, "R": _log(rng, 1, 16384), "d": _log(rng, 16, 2048), "V": _log(rng, 2, 131072),
                 "train": rng.random() < 0.7, "skip": rng.choice((0.0, 0.1, 0.5))}
            if c["R"] * c["d"] * c["V"] * (4 if c["train"] else 1) <= 8192 * 1024 * 50001 * 4:
                return c
    if op == "head":
        while True:
            D = rng.choice((32, 48, 64, 80, 96, 128, 192, 256))
            c = {"op": op, "B": _log(rng, 1, 512), "T": _log(rng, 1, 8192), "H": _log(rng, 1, 32), "D": D,
                 "rotary": rng.choice((D, D // 2)), "interleaved": rng.random() < 0.4, "shared": rng.random() < 0.6,
                 "start": rng.choice((0, 1000, 1000000)), "train": rng.random() < 0.7}
            if c["B"] * c["T"] * c["H"] * D <= 2 * 8191 * 32 * 128:
                return c
    while True:
        c = {"op": op, "B": _log(rng, 1, 16), "m": _log(rng, 16, 4096), "n": _log(rng, 16, 4096)}
        if _orth_flops(c) <= 5 * 4 * 4096 ** 3:
            return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=g).mul_(std)


def _nll_inputs(c, seed):
    g = _gen(seed)
    R, d, V = c["R"], c["d"], c["V"]
    t = {"h": _normal(g, R, d), "w": _normal(g, d, V, std=2 / math.sqrt(d)), "b": _normal(g, V, std=0.1),
         "t": torch.randint(0, V, (R,), device="cuda", generator=g).float()}
    if c["skip"]:
        t["t"][torch.rand(R, device="cuda", generator=g) < c["skip"]] = -1.0
    if c["train"]:   # a mean over the rows that count, as the loss's gradient hands it down
        t["gy"] = (t["t"] >= 0).float() / (t["t"] >= 0).sum().clamp(min=1)
    return t


def _head_inputs(c, seed):
    g = _gen(seed)
    B, T, H, D = c["B"], c["T"], c["H"], c["D"]
    t = {"x": _normal(g, B, T, H, D), "gain": 1 + _normal(g, D, std=0.1)}
    pos = torch.arange(T, device="cuda", dtype=torch.float32) + c["start"]
    if not c["shared"]:   # every sequence of the batch starts at a place of its own
        pos = pos + torch.randint(0, 1000, (B, 1), device="cuda", generator=g)
    t["pos"] = pos.contiguous()
    if c["train"]:
        t["gy"] = _normal(g, B, H, T, D)
    return t


def _orth_inputs(c, seed):
    g = _gen(seed)
    # a momentum buffer: noise over a few strong directions
    B, m, n = c["B"], c["m"], c["n"]
    k = min(8, m, n)
    x = _normal(g, B, m, n) + 3 * torch.matmul(_normal(g, B, m, k), _normal(g, B, k, n)) / math.sqrt(k)
    return {"x": (x * 1e-3).contiguous()}


def prepare(case, seed):
    t = {"nll": _nll_inputs, "head": _head_inputs, "orth": _orth_inputs}[case["op"]](case, seed)
    s = {"case": case, "in": t}
    if own:
        s["program"], s["out"] = _program(case, t)
    return s


# ---------------------------------------------------------------- the plain form
def _nll_plain(c, t):
    h, w, gy = t["h"], t["w"], t.get("gy")
    keep = t["t"] >= 0
    idx = t["t"].clamp(min=0).long()[:, None]
    z = torch.matmul(h, w) + t["b"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    nll = torch.where(keep, (torch.log(total) - z.gather(1, idx))[:, 0], 0.0)
    if gy is None:
        return {"nll": nll}
    del z
    g = torch.where(keep, gy, 0.0)[:, None]
    dz = e.mul_(g / total)
    dz.scatter_add_(1, idx, -g)
    return {"nll": nll, "dh": torch.matmul(dz, w.t()), "dw": torch.matmul(h.t(), dz), "db": dz.sum(0)}


def _rotations(c, pos, dtype):
    """cos and sin [B or 1, T, 1, rotary / 2] of every position's angles, in 64 bits until the end."""
    k = c["rotary"] // 2
    inv = 10000.0 ** (-torch.arange(k, device=pos.device, dtype=torch.float64) / k)
    a = pos.double().reshape(-1, c["T"], 1, 1) * inv
    return torch.cos(a).to(dtype), torch.sin(a).to(dtype)


def _rotate(c, x, cos, sin):
    r, k = c["rotary"], c["rotary"] // 2
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :k], x[..., k:r]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return y if r == c["D"] else torch.cat((y, x[..., r:]), -1)


def _head_forms(c, t, dtype):
    x, gain = t["x"].to(dtype), t["gain"].to(dtype)
    cos, sin = _rotations(c, t["pos"], dtype)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS_ROOT)
    n = x * r
    out = {"y": _rotate(c, n * gain, cos, sin).transpose(1, 2).contiguous()}
    if c["train"]:
        u = _rotate(c, t["gy"].to(dtype).transpose(1, 2), cos, -sin)
        out["dgain"] = (u * n).sum((0, 1, 2))
        u = u * gain
        out["dx"] = r * (u - n * (u * n).mean(-1, keepdim=True))
    return out


def _orth_forms(c, x, dtype):
    a, b, k = NS
    x = x.to(dtype)
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + EPS_NORM)
    tall = c["m"] > c["n"]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(5):
        s = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * s + k * torch.matmul(s, s), x)
    return {"o": (x.transpose(-2, -1) if tall else x).contiguous()}


def run(state):
    c, t = state["case"], state["in"]
    if own:
        state["program"].run()
        return state["out"]
    if c["op"] == "nll":
        return _nll_plain(c, t)
    if c["op"] == "head":
        return _head_forms(c, t, torch.float32)
    return _orth_forms(c, t["x"], torch.float32)


# ---------------------------------------------------------------- the framework's operators
_runner = None


def _program(c, t):
    """The resident program of one case, reading its inputs and writing its outputs in place."""
    global _runner
    pkg = importlib.import_module(PKG)
    rt = importlib.import_module(PKG + ".runtime")
    cg = importlib.import_module(PKG + ".codegen")
    if _runner is None:
        _runner = rt.GpuRunner.create(torch.cuda.current_device())
    g = pkg.ir.Graph()
    ids = {k: g.input(k, list(v.shape)) for k, v in t.items() if k != "gy"}
    if c["op"] == "nll":
        out = {"nll": g.linear_nll(ids["h"], ids["w"], ids["b"], ids["t"])}
        wrt = {"dh": ids["h"], "dw": ids["w"], "db": ids["b"]}
    elif c["op"] == "head":
        out = {"y": g.head_norm_rope(ids["x"], ids["gain"], ids["pos"], rotary=c["rotary"],
                                     interleaved=c["interleaved"], eps=EPS_ROOT)}
        wrt = {"dx": ids["x"], "dgain": ids["gain"]}
    else:
        out = {"o": g.orthogonalize(ids["x"], steps=5, coeffs=NS, eps=EPS_NORM)}
        wrt = {}
    if "gy" in t:
        G = pkg.autodiff.grad(g, list(out.values()), list(wrt.values()))
        g = G.graph
        out.update(zip(wrt, G.grads))
        ids["gy"] = g.input_id(G.cotangents[0])
    f = pkg.fuse.fuse(g, keep=list(out.values()))
    lowered = cg.lower_fused(f.graph, matmul="tiled", keep=[f.index[i] for i in out.values()])
    place = {f.index[ids[k]]: v.data_ptr() for k, v in t.items()}
    made = {}
    for k, i in out.items():
        made[k] = torch.empty(g.shape(i), device="cuda")
        place[f.index[i]] = made[k].data_ptr()
    torch.cuda.synchronize()
    _runner.set_stream(0)            # captured on the runner's own stream, replayed on torch's
    program = rt.Program(_runner, f.graph, lowered, keep=[f.index[i] for i in out.values()], place=place,
                         batch=True, capture=True)
    _runner.sync()
    _runner.set_stream(torch.cuda.current_stream().cuda_stream or 1)   # 1: the legacy default stream
    return program, made


# ---------------------------------------------------------------- work and the answer in 64 bits
def _orth_flops(c):
    m, n = min(c["m"], c["n"]), max(c["m"], c["n"])
    return 5 * c["B"] * (m * m * n + m ** 3 + 2 * m * m * n)   # both symmetric products need one half only


def work(case):
    c = case
    if c["op"] == "nll":
        R, d, V = c["R"], c["d"], c["V"]
        n = R * d + d * V + V + 2 * R
        flops = 2 * R * d * V
        if c["train"]:
            n += R + R * d + d * V + V
            flops *= 3
        return {"bytes": 4 * n, "flops": flops}
    if c["op"] == "head":
        e = c["B"] * c["T"] * c["H"] * c["D"]
        return {"bytes": 4 * e * (5 if c["train"] else 2), "flops": e * (25 if c["train"] else 9)}
    return {"bytes": 8 * c["B"] * c["m"] * c["n"], "flops": _orth_flops(c)}


def exact(case, seed):
    c = case
    if c["op"] == "head":
        return _head_exact(c, _head_inputs(c, seed))
    if c["op"] == "nll":
        return _nll_exact(c, _nll_inputs(c, seed))
    return _orth_exact(c, _orth_inputs(c, seed)["x"])


def _nll_exact(c, t):
    """A block of rows at a time, in 64 bits."""
    R, V, w = c["R"], c["V"], t["w"].double()
    nll = torch.zeros(R, device="cuda", dtype=torch.float64)
    dh = torch.zeros(R, c["d"], device="cuda", dtype=torch.float64)
    dw, db = torch.zeros_like(w), torch.zeros(V, device="cuda", dtype=torch.float64)
    step = max(1, (1 << 28) // V)
    for i in range(0, R, step):
        h, idx = t["h"][i:i + step].double(), t["t"][i:i + step].long()
        rows = (idx >= 0).nonzero()[:, 0]
        if not len(rows):
            continue
        h, idx = h[rows], idx[rows]
        logp = torch.log_softmax(h @ w + t["b"].double(), 1)
        at = torch.arange(len(rows), device="cuda")
        nll[i + rows] = -logp[at, idx]
        if c["train"]:
            p = logp.exp_()
            p[at, idx] -= 1
            p *= t["gy"][i:i + step][rows].double()[:, None]
            dh[i + rows] = p @ w.t()
            dw += h.t() @ p
            db += p.sum(0)
    return {"nll": nll, "dh": dh, "dw": dw, "db": db} if c["train"] else {"nll": nll}


def _head_exact(c, t):
    """One 2 x 2 turn at a time as complex numbers, the gradients from torch's autograd, in 64 bits."""
    x = t["x"].double().requires_grad_(c["train"])
    gain = t["gain"].double().requires_grad_(c["train"])
    k, r = c["rotary"] // 2, c["rotary"]
    freq = torch.exp(-math.log(10000.0) * torch.arange(k, device="cuda", dtype=torch.float64) / k)
    angle = t["pos"].double().view(-1, c["T"])[:, :, None, None] * freq
    turn = torch.polar(torch.ones_like(angle), angle)
    n = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["D"] + EPS_ROOT) * gain
    pairs = n[..., :r].unflatten(-1, (k, 2)) if c["interleaved"] else n[..., :r].unflatten(-1, (2, k)).transpose(-1, -2)
    q = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    q = q.flatten(-2) if c["interleaved"] else q.transpose(-1, -2).flatten(-2)
    y = torch.cat((q, n[..., r:]), -1).permute(0, 2, 1, 3)
    out = {"y": y.detach().contiguous()}
    if c["train"]:
        out["dx"], out["dgain"] = torch.autograd.grad(y, (x, gain), t["gy"].double())
    return out


def _orth_exact(c, x):
    """By the Gram matrix alone, in 64 bits: with S = X X^T every step multiplies X by P = a + b S + c S S,
    which commutes with S, so S becomes P S P and the P's can be multiplied together first."""
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS_NORM)
    wide = c["m"] <= c["n"]
    s = x @ x.mT if wide else x.mT @ x
    eye = torch.eye(s.shape[-1], device="cuda", dtype=torch.float64)
    q = eye
    for _ in range(5):
        p = NS[0] * eye + s @ (NS[1] * eye + NS[2] * s)
        q, s = q @ p, p @ s @ p
    return {"o": q @ x if wide else x @ q}
