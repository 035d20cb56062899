// lower_training.h -- launches of the operators of a decoder's training step (linearNll, headNormRope, their
// gradients, orthogonalize), the records that the Python host's training_ops.py makes, field for field.
// Part of lower.cpp (it uses that file's helpers); graphs arrive as JSON, so the shapes and attributes that
// a kernel's addresses follow from are checked here as the Python host's IR checks them.
#pragma once

static std::string to_json(const Value& v);

static bool is_training(const std::string& op) {
  return op == "linearNll" || op == "linearNllGrad" || op == "headNormRope" || op == "headNormRopeGrad" ||
         op == "orthogonalize";
}

constexpr i64 F16_FLAG = (i64)1 << 33, PAIR_FLAG = (i64)1 << 34;
constexpr i64 F16_BM = 128, F16_BK = 32;
constexpr i64 F16_EXTRA = 256 + 8 * 128 + 8 * 4096 + 1024;
constexpr i64 AMAX_BLOCKS = 4 * SM_COUNT, DZ_BYTES = (i64)128 << 20;
constexpr i64 CTRL_BYTES = 4 * (4 + 8 * 2 * SM_COUNT);
constexpr i64 JOIN_COUNTERS = 512, JOIN_PARTS = 4, NLL_CTRL_BYTES = CTRL_BYTES + 4 * JOIN_COUNTERS;
constexpr i64 NLL_CHUNK = 256, NS_CHUNK = 128, NS_PARTS = 512;
constexpr i64 NLL_ROWS = 16;
constexpr i64 NLL_ADD = 1, NLL_JOIN = 2, NLL_NO_LOSS = 4, NLL_DB = 8;
constexpr double F16_ROOM = 60000.0;
constexpr i64 MAX_DIM = (i64)1 << 30, MAX_VALUES = (i64)1 << 40;

static i64 up_to(i64 n, i64 k) { return cdiv(n, k) * k; }
static i64 nll_pitch(i64 cols) { return std::min<i64>(256, up_to(cols, 32)); }

[[noreturn]] static void refuse(const Node& n, const std::string& what) {
  throw Error("node " + std::to_string(n.id) + " (" + n.op + "): " + what);
}
static const Value& attr(const Node& n, const std::string& name) {
  const Value* v = n.attrs_json.find(name);
  if (!v) refuse(n, "no attribute '" + name + "'");
  return *v;
}
static bool bool_attr(const Node& n, const std::string& name) {
  const Value& v = attr(n, name);
  if (v.kind != Value::Bool) refuse(n, name + " must be true or false");
  return v.b;
}
static double number_attr(const Node& n, const std::string& name) {
  const Value& v = attr(n, name);
  if (!v.is_number() || !std::isfinite(v.num)) refuse(n, name + " must be a number");
  return v.num;
}
static i64 int_attr(const Node& n, const std::string& name) {
  const Value& v = attr(n, name);
  if (!v.is_number() || !v.integral) refuse(n, name + " must be an integer");
  return v.as_int();
}
static std::string word_attr(const Node& n, const std::string& name) {
  const Value* v = n.attrs_json.find(name);
  return v && v->is_string() ? v->str : "";
}
static void expect(const Node& n, bool ok, const std::string& what) {
  if (!ok) refuse(n, what);
}
// eps as the kernel takes it, a float32: one above 0 must stay so, or a zero norm is divided by zero.
static void check_eps(const Node& n) {
  const double eps = number_attr(n, "eps");
  expect(n, eps >= 0 && std::isfinite((float)eps) && (eps == 0 || (float)eps > 0),
         "eps must be 0 or a positive float32");
}
static const std::vector<i64>& in_shape(const Graph& g, const Node& n, size_t k) {
  expect(n, k < n.inputs.size(), "too few inputs");
  return g.nodes[n.inputs[k]].shape;
}
using Shape = std::vector<i64>;

struct NllSaved { i64 lse, h, w, floats; };
static NllSaved nll_saved(i64 R, i64 d, i64 V) {
  auto blocked = [](i64 n) { return n <= 256 ? up_to(n, 32) : up_to(n, 256); };
  NllSaved s;
  s.lse = up_to(256 + 4 * up_to(V, 256), 256);
  s.h = up_to(s.lse + 8 * R, 256);
  s.w = up_to(s.h + 4 * R * blocked(d), 256);
  s.floats = up_to(s.w + 4 * d * blocked(V), 256) / 4;
  return s;
}

static void newton_schulz_scales(const Node& n, i64 steps, const double co[3], int out[3]) {
  const double a = co[0], b = co[1], c = co[2];
  double top = 1.0, mx = 0.0, ms = 0.0, mp = 0.0;
  for (i64 k = 0; k < steps; ++k) {
    double s = top * top;
    mx = std::max(mx, top);
    ms = std::max(ms, s);
    mp = std::max(mp, std::fabs(b * s + c * s * s));
    if (c != 0 && 0 < -b / (2 * c) && -b / (2 * c) < s) mp = std::max(mp, std::fabs(b * b / (4 * c)));
    double nxt = std::fabs(a * top + b * top * s + c * top * s * s);
    std::vector<double> roots;
    if (c != 0) {
      double disc = 9 * b * b - 20 * a * c;
      if (disc >= 0) roots = {(-3 * b + std::sqrt(disc)) / (10 * c), (-3 * b - std::sqrt(disc)) / (10 * c)};
    } else if (b != 0) {
      roots = {-a / (3 * b)};
    }
    for (double t : roots)
      if (0 < t && t < s) {
        double q = std::sqrt(t);
        nxt = std::max(nxt, std::fabs(a * q + b * q * t + c * q * t * t));
      }
    top = nxt * 1.01;
  }
  const double bounds[3] = {mx, ms, mp};
  for (int i = 0; i < 3; ++i) {
    int k = 0;
    while (k < 15 && bounds[i] * 1.01 * (2 << k) <= F16_ROOM) ++k;
    if (!(bounds[i] * 1.01 * (1 << k) <= F16_ROOM)) refuse(n, "coefficients let the values grow beyond fp16");
    out[i] = k;
  }
}

// Shapes and attributes, as the Python host's infer_shape checks them.
static void check_training(const Graph& g, const Node& n) {
  for (size_t k = 0; k < n.inputs.size(); ++k) {
    // (the saved value of linearNllGrad has one axis of any length)
    const i64 most = n.op == "linearNllGrad" && k == 1 ? MAX_VALUES : MAX_DIM;
    i64 values = 1;
    for (i64 d : g.nodes[n.inputs[k]].shape) {
      expect(n, d >= 1, "operand of an empty shape");
      expect(n, d <= most && values <= MAX_VALUES / d, "operand beyond 2^30 an axis or 2^40 values");
      values *= d;
    }
  }
  Shape want;
  if (n.op == "linearNll") {
    const bool bias = bool_attr(n, "bias");
    expect(n, n.inputs.size() == 3u + bias, "wrong number of inputs");
    const Shape &h = in_shape(g, n, 0), &w = in_shape(g, n, 1);
    expect(n, h.size() == 2 && w.size() == 2 && h[1] == w[0], "rows and weight must be [R,d] and [d,V]");
    expect(n, w[1] <= ((i64)1 << 24), "too many classes");
    expect(n, !bias || in_shape(g, n, 2) == Shape{w[1]}, "bias of another shape");
    expect(n, in_shape(g, n, 2 + bias) == Shape{h[0]}, "targets of another shape");
    const std::string out = word_attr(n, "out");
    expect(n, out == "loss" || out == "saved", "out must be 'loss' or 'saved'");
    want = out == "loss" ? Shape{h[0]} : Shape{nll_saved(h[0], w[0], w[1]).floats};
  } else if (n.op == "linearNllGrad") {
    const bool bias = bool_attr(n, "bias");
    expect(n, n.inputs.size() == 3, "wrong number of inputs");
    const i64 d = int_attr(n, "d"), V = int_attr(n, "V");
    expect(n, d >= 1 && d <= MAX_DIM && V >= 1 && V <= ((i64)1 << 24), "d and V must be the weight's sizes");
    const Shape& t = in_shape(g, n, 0);
    expect(n, t.size() == 1 && in_shape(g, n, 2) == t && in_shape(g, n, 1) == Shape{nll_saved(t[0], d, V).floats},
           "targets, saved value and cotangent do not belong together");
    const std::string wrt = word_attr(n, "wrt");
    expect(n, wrt == "h" || wrt == "w" || (wrt == "b" && bias), "no such gradient");
    want = wrt == "h" ? Shape{t[0], d} : wrt == "w" ? Shape{d, V} : Shape{V};
  } else if (n.op == "headNormRope" || n.op == "headNormRopeGrad") {
    const bool back = n.op == "headNormRopeGrad";
    expect(n, n.inputs.size() == 3u + back, "wrong number of inputs");
    const Shape &x = in_shape(g, n, 0), &pos = in_shape(g, n, 2);
    expect(n, x.size() == 4 && x[3] <= 512, "x must be [B,T,H,D], D at most 512");
    expect(n, in_shape(g, n, 1) == Shape{x[3]}, "gain of another shape");
    const Shape shared{x[1]}, each{x[0], x[1]};
    expect(n, pos == shared || pos == each, "positions must be [T] or [B,T]");
    const i64 r = int_attr(n, "rotary");
    expect(n, r >= 0 && r <= x[3] && r % 2 == 0, "rotary must be an even part of a head");
    bool_attr(n, "interleaved");
    check_eps(n);
    expect(n, number_attr(n, "base") > 0, "base must be a number above 0");
    const Shape y = bool_attr(n, "headsFirst") ? Shape{x[0], x[2], x[1], x[3]} : x;
    if (back) {
      expect(n, in_shape(g, n, 3) == y, "cotangent of another shape");
      const std::string wrt = word_attr(n, "wrt");
      expect(n, wrt == "x" || wrt == "gain", "no such gradient");
      want = wrt == "x" ? x : Shape{x[3]};
    } else {
      want = y;
    }
  } else {
    expect(n, n.inputs.size() == 1, "wrong number of inputs");
    const Shape& x = in_shape(g, n, 0);
    expect(n, x.size() >= 2, "needs rank >= 2");
    i64 batch = 1;
    for (size_t k = 0; k + 2 < x.size(); ++k) batch *= x[k];
    expect(n, batch <= 65535, "too many matrices");
    const i64 steps = int_attr(n, "steps");
    expect(n, steps >= 1 && steps <= 32, "steps must be 1 to 32");
    const Value& co = attr(n, "coeffs");
    expect(n, co.is_array() && co.arr.size() == 3, "coeffs must be three numbers");
    for (auto& v : co.arr)
      expect(n, v.is_number() && std::isfinite((float)v.num), "coeffs must be three float32 numbers");
    check_eps(n);
    const double c[3] = {co.arr[0].num, co.arr[1].num, co.arr[2].num};
    int k[3];
    newton_schulz_scales(n, steps, c, k);
    want = x;
  }
  expect(n, n.shape == want, "stored shape is not the inferred one");
}

// {node: the nodes of its launch}: outputs of one launch differ in which output they are only.
static std::map<int, std::vector<int>> siblings(const Graph& g) {
  std::map<std::string, std::vector<std::vector<int>>> groups;
  std::map<int, std::pair<std::string, size_t>> of;
  auto which = [&](const Node& n) {
    std::string w = word_attr(n, "wrt");
    return w.empty() ? word_attr(n, "out") : w;
  };
  for (auto& n : g.nodes) {
    if (!is_training(n.op) || which(n).empty()) continue;
    std::map<std::string, std::string> rest;
    for (auto& kv : n.attrs_json.obj)
      if (kv.first != "wrt" && kv.first != "out") rest[kv.first] = to_json(kv.second);
    std::string key = n.op;
    for (int i : n.inputs) key += "," + std::to_string(i);
    for (auto& kv : rest) key += ";" + kv.first + "=" + kv.second;
    auto& gs = groups[key];
    size_t k = 0;
    for (; k < gs.size(); ++k) {
      bool has = false;
      for (int i : gs[k]) has |= which(g.nodes[i]) == which(n);
      if (!has) break;
    }
    if (k == gs.size()) gs.emplace_back();
    gs[k].push_back(n.id);
    of[n.id] = {key, k};
  }
  std::map<int, std::vector<int>> out;
  for (auto& kv : of) out[kv.first] = groups[kv.second.first][kv.second.second];
  return out;
}

// ---------------------------------------------------------------- split-fp16 products
struct Tile {   // of a product: ctas * 128 rows x bn columns
  i64 bn = 0, ctas = 1;
  i64 cols() const { return bn / ctas; }   // of B, loaded by one CTA
  std::string name() const { return std::to_string(bn) + (ctas == 2 ? "x2" : ""); }
};
static i64 f16_smem(const Tile& t) {
  i64 stage = 2 * F16_BM * F16_BK * 2 + 2 * t.cols() * F16_BK * 2;
  i64 stages = std::min<i64>(8, (227 * 1024 - F16_EXTRA) / stage);
  return stages * stage + F16_EXTRA;
}
static i64 f16_tiles(i64 M, i64 N, const Tile& tile, bool symmetric) {
  const i64 rows = F16_BM * tile.ctas;
  i64 tm = cdiv(M, rows), tn = cdiv(N, tile.bn), t = 0;
  if (!symmetric) return tm * tn;
  for (i64 i = 0; i < tm; ++i) t += tn - i * rows / tile.bn;
  return t;
}

struct F16Plan {
  Tile tile;
  i64 grid = 0, whole = 0, quantum = 0;
};
static F16Plan f16_plan(i64 M, i64 N, i64 K, i64 batch, i64 chunk, bool symmetric = false, const Tile* only = nullptr) {
  static const i64 COST[4][6] = {{256, 2, 275, 6600, 3000, 2500}, {128, 2, 173, 3600, 1500, 1600},
                                 {128, 1, 180, 3000, 1500, 1200}, {64, 1, 140, 1500, 1000, 700}};
  F16Plan best;
  i64 cost = -1;
  auto take = [&](i64 c, const Tile& tile, i64 grid, i64 whole, i64 q) {
    if (cost >= 0 && c >= cost) return;
    cost = c;
    best = {tile, grid, whole, q};
  };
  const i64 steps = cdiv(K, 16);
  for (auto& row : COST) {
    const Tile tile{row[0], row[1]};
    const i64 step = row[2], epi = row[3], once = row[4], part = row[5], units = SM_COUNT / tile.ctas;
    if (only ? tile.bn != only->bn || tile.ctas != only->ctas
             : (tile.bn > 64 && N <= tile.bn / 2) || M <= F16_BM * (tile.ctas - 1))
      continue;
    const i64 tiles = batch * f16_tiles(M, N, tile, symmetric);
    take(cdiv(tiles, units) * (steps * step + epi), tile, std::min<i64>(units, tiles) * tile.ctas, tiles, 1);
    for (i64 q = 1; q <= 64; q *= 2) {
      const i64 per = cdiv(K, 256 * q);
      if (only || tiles >= units || per == 1) break;
      const i64 grid = std::min<i64>(units, tiles * per), run = cdiv(tiles * per, grid);
      const i64 pieces = run == 1 ? per : per / run + 2;
      take(run * q * 16 * step + once + pieces * part + epi, tile, grid * tile.ctas, 0, q * (256 / chunk));
    }
  }
  return best;
}
static i64 f16_partial_bytes(const F16Plan& p, i64 tiles) { return p.whole == tiles ? 0 : 2 * p.grid * F16_BM * p.tile.bn * 4; }

static Map f16_operand(i64 off, i64 cols, i64 rows, i64 batch, i64 pitch, bool mn, i64 box_rows) {
  return {"scratch", off, cols, rows, 2 * batch, pitch * 2, rows * pitch * 2, (mn ? 64 : F16_BK) | F16_FLAG | PAIR_FLAG,
          mn ? F16_BK : box_rows};
}
static Map blocked(const std::string& region, i64 off, i64 rows, i64 cols, i64 pitch, i64 box_cols, i64 box_rows) {
  return {region, off, pitch, rows, 2 * cdiv(cols, 256), pitch * 2, rows * pitch * 2, box_cols | F16_FLAG | PAIR_FLAG, box_rows};
}
static Map blocked_operand(const std::string& region, i64 off, i64 rows, i64 cols, i64 pitch, bool mn, i64 box_rows) {
  return mn ? blocked(region, off, rows, cols, pitch, 64, F16_BK)
            : blocked(region, off, rows, cols, pitch, F16_BK, box_rows);
}

static Call f16_gemm(const std::string& name, i64 M, i64 N, i64 K, i64 batch, const F16Plan& p, i64 part_at,
                     std::vector<Map> maps, const std::vector<i64>& params, i64 err, i64* partial, bool symmetric = false) {
  const i64 tiles = batch * f16_tiles(M, N, p.tile, symmetric);
  if (tiles >= ((i64)1 << 31)) throw Error(name + ": " + std::to_string(tiles) + " tiles");
  std::vector<i64> ps = {M | N << 32, K | batch << 32, p.whole | p.quantum << 32, part_at};
  ps.insert(ps.end(), params.begin(), params.end());
  Call c = make_call(name + "_" + p.tile.name(), {p.grid, 1, 1}, {384, 1, 1}, f16_smem(p.tile), ps);
  c.tma = std::move(maps);
  c.has_tma = true;
  c.err_offset = err;
  *partial = f16_partial_bytes(p, tiles);
  return c;
}

// Scratch regions one behind the other.
struct Regions {
  i64 end = 0;
  i64 add(i64 nbytes) {
    i64 at = end;
    end += up_to(nbytes, 256);
    return at;
  }
};

static Launch training_record(const Node& n, const std::string& kind, std::string code, std::vector<Call> calls, i64 scratch) {
  Launch l;
  l.node = n.id;
  l.op = n.op;
  l.kind = kind;
  l.inputs = n.inputs;
  l.code = std::move(code);
  l.calls = std::move(calls);
  l.scratch_bytes = scratch;
  return l;
}

// ---------------------------------------------------------------- linearNll
static bool nll_joined(i64 groups, i64 parts) { return groups <= JOIN_COUNTERS && parts <= JOIN_PARTS; }
static std::string nll_source(bool bias) {
  return std::string("// cross entropy of a linear head, ") + (bias ? "bias" : "no bias") + "\n#include \"tcb/common.cuh\"\n#define TCB_BIAS " +
         (bias ? "1" : "0") + "\n#include \"tcb/linear_nll.cuh\"\n";
}
static std::vector<i64> cat(std::vector<i64> a, const std::vector<i64>& b) {
  a.insert(a.end(), b.begin(), b.end());
  return a;
}

// A few rows' loss alone (tcb/nll_rows.cuh).
static Launch nll_rows_launch(const Graph& g, const Node& node, i64 R, i64 d, i64 V) {
  const i64 rows = R <= 4 ? 4 : R <= 8 ? 8 : 16, blocks = cdiv(V, 128);
  i64 parts = std::min<i64>({8, std::max<i64>(1, 4 * SM_COUNT / blocks), cdiv(d, 64)});
  const i64 per = cdiv(d, parts);
  parts = cdiv(d, per);
  Regions r;
  r.add(parts > 1 ? 4 * parts * R * V : 0);
  const i64 zt = r.add(4 * R), stats = r.add(8 * R * cdiv(V, 32));
  const std::vector<i64> params = {parts, per, zt, stats, R, d, V};
  std::vector<Call> calls = {make_call("tcb_nll_rows_" + std::to_string(rows), {blocks, parts, 1}, {256, 1, 1}, 0, params)};
  if (parts > 1) calls.push_back(make_call("tcb_nll_rows_add", {cdiv(V, 256), R, 1}, {256, 1, 1}, 0, params));
  calls.push_back(make_call("tcb_nll_rows_finish", {R, 1, 1}, {1024, 1, 1}, 0, params));
  std::string code = nll_source(bool_attr(node, "bias"));
  code.replace(code.find("linear_nll.cuh"), 14, "nll_rows.cuh");
  Launch l = training_record(node, "linear-nll", code, std::move(calls), r.end);
  l.info = {{"rnv", arr({num(R), num(d), num(V)})}, {"parts", num(parts)}, {"path", str("fma")}};
  return l;
}

static Launch nll_launch(const Graph& g, const std::vector<int>& ids) {
  const Node& node = g.nodes[ids[0]];
  const i64 R = in_shape(g, node, 0)[0], d = in_shape(g, node, 0)[1], V = in_shape(g, node, 1)[1];
  int loss = -1, saved = -1;
  for (int i : ids) (word_attr(g.nodes[i], "out") == "loss" ? loss : saved) = i;
  if (saved < 0 && R <= NLL_ROWS) return nll_rows_launch(g, node, R, d, V);
  const NllSaved in = nll_saved(R, d, V);
  const F16Plan plan = f16_plan(R, V, d, 1, NLL_CHUNK);
  const i64 halves = cdiv(V, plan.tile.bn / 2);
  Regions r;
  r.add(8 * AMAX_BLOCKS);
  const i64 err = r.add(NLL_CTRL_BYTES), zt = r.add(4 * R), part = r.add(8 * R * halves);
  r.add(loss >= 0 ? 0 : 4 * R);
  const i64 saved_at = r.add(saved >= 0 ? 0 : 4 * in.floats);
  const bool joined = nll_joined(cdiv(R, 32), halves);
  const std::vector<i64> tail = {R, d, V, saved_at, in.lse, in.h, in.w, zt, part,
                                 (joined ? NLL_JOIN : 0) | (loss >= 0 ? 0 : NLL_NO_LOSS)};
  const std::string region = saved >= 0 ? "out" : "scratch";
  const i64 base = saved >= 0 ? 0 : saved_at;
  std::vector<Map> maps = {blocked_operand(region, base + in.h, R, d, nll_pitch(d), false, F16_BM),
                           blocked_operand(region, base + in.w, d, V, nll_pitch(V), true, plan.tile.cols())};
  const i64 blocks = std::max<i64>(1, std::min<i64>(AMAX_BLOCKS, cdiv(R * d + d * V, 2048)));
  const i64 units = d * cdiv(V, 1024) + R * cdiv(d, 1024);
  i64 partial = 0;
  std::vector<Call> calls;
  calls.push_back(make_call("tcb_nll_amax", {blocks, 1, 1}, {256, 1, 1}, 0, cat({blocks, 0, 0, 0}, tail)));
  calls[0].err_offset = err;
  calls.push_back(make_call("tcb_nll_split", {std::max<i64>(2, std::min<i64>(units, SM_COUNT * 8)), 1, 1}, {256, 1, 1}, 0,
                            cat({blocks, 0, 0, 0}, tail)));
  calls.push_back(f16_gemm("tcb_nll_logits", R, V, d, 1, plan, r.end, maps, tail, err, &partial));
  if (!joined)
    calls.push_back(make_call("tcb_nll_finish", {cdiv(R, 32), 1, 1}, {256, 1, 1}, 0, cat({halves, 0, 0, 0}, tail)));
  if (saved >= 0)
    for (auto& c : calls) {
      c.ptr_params = {{14, saved}};
      if (loss >= 0) c.ptr_params.push_back({7, loss});
      if (saved != node.id) c.out_node = saved;
    }
  Launch l = training_record(node, "linear-nll", nll_source(bool_attr(node, "bias")), std::move(calls),
                             r.end + up_to(partial, 256));
  l.info = {{"rnv", arr({num(R), num(d), num(V)})}, {"tile", str(plan.tile.name())}, {"ctrl_bytes", num(up_to(NLL_CTRL_BYTES, 64))},
            {"path", str("tcgen05-f16x3")}};
  return l;
}

static Launch nll_grad_launch(const Graph& g, const std::vector<int>& ids) {
  const Node& node = g.nodes[ids[0]];
  const i64 R = in_shape(g, node, 0)[0], d = int_attr(node, "d"), V = int_attr(node, "V");
  const NllSaved in = nll_saved(R, d, V);
  const F16Plan fwd = f16_plan(R, V, d, 1, NLL_CHUNK);
  const i64 most = std::max<i64>(256, DZ_BYTES / (4 * R) / 256 * 256);
  const i64 piece = std::min<i64>(up_to(cdiv(V, cdiv(V, most)), 256), up_to(V, 32)), pieces = cdiv(V, piece);
  std::map<std::string, int> want;
  for (int i : ids) want[word_attr(g.nodes[i], "wrt")] = i;
  const bool wh = want.count("h"), ww = want.count("w"), wb = want.count("b");
  Regions r;
  r.add(256);
  const i64 err = r.add(NLL_CTRL_BYTES), dz = r.add(4 * R * up_to(piece, piece > 256 ? 256 : 32)),
            db = r.add(wb ? 4 * cdiv(R, 32) * V : 0);
  const std::vector<i64> tail = {R, d, V, 0, in.lse, in.h, in.w, db};
  const bool joined = wb && nll_joined(cdiv(V, 32), cdiv(R, 32));
  std::vector<Call> calls;
  calls.push_back(make_call("tcb_gemm_prep", {1, 1, 1}, {128, 1, 1}));
  calls[0].err_offset = err;
  i64 partial = 0;
  auto to = [&](Call& c, const std::string& wrt) {
    if (want[wrt] != node.id) c.out_node = want[wrt];
  };
  for (i64 k = 0; k < pieces; ++k) {
    const i64 v0 = k * piece, n = std::min(piece, V - v0);
    const std::vector<i64> params = cat(tail, {v0, (k ? NLL_ADD : 0) | (joined ? NLL_JOIN : 0) | (wb ? NLL_DB : 0)});
    const i64 w_at = in.w + (v0 ? 4 * d * v0 : 0);
    auto h = [&](bool mn) { return blocked_operand("in_at", in.h << 3 | 1, R, d, nll_pitch(d), mn, F16_BM); };
    auto w = [&](bool mn, i64 box_rows) { return blocked_operand("in_at", w_at << 3 | 1, d, n, nll_pitch(V), mn, box_rows); };
    auto z = [&](bool mn, i64 box_rows) { return blocked_operand("scratch", dz, R, n, nll_pitch(n), mn, box_rows); };
    auto add = [&](const std::string& name, i64 M, i64 N, i64 K, const F16Plan& p, std::vector<Map> maps) -> Call& {
      i64 nbytes = 0;
      calls.push_back(f16_gemm(name, M, N, K, 1, p, r.end, std::move(maps), params, err, &nbytes));
      partial = std::max(partial, nbytes);
      return calls.back();
    };
    // the forward's own plan, or its tile
    const F16Plan pz = pieces == 1 ? fwd : f16_plan(R, n, d, 1, NLL_CHUNK, false, &fwd.tile);
    Call& c = add("tcb_nll_dz", R, n, d, pz, {h(false), w(true, pz.tile.cols()), blocked("scratch", dz, R, n, nll_pitch(n), 32, 32)});
    if (joined) c.ptr_params = {{14, want["b"]}};
    const F16Plan ph = f16_plan(R, d, n, 1, NLL_CHUNK), pw = f16_plan(d, n, R, 1, NLL_CHUNK);
    if (wh && ww && ph.tile.ctas == 1 && pw.tile.ctas == 1 && ph.grid + pw.grid <= SM_COUNT) {
      i64 hb = 0;
      Call b = f16_gemm("tcb_nll_both", R, d, n, 1, ph, r.end, {z(false, F16_BM), w(false, ph.tile.cols()), h(true), z(true, pw.tile.cols())}, params, err, &hb);
      b.name = "tcb_nll_both_" + ph.tile.name() + "_" + pw.tile.name();
      b.grid[0] = ph.grid + pw.grid;
      b.smem = std::max(f16_smem(ph.tile), f16_smem(pw.tile));
      b.params[7] = pw.whole | pw.quantum << 32;
      b.params[8] = r.end + up_to(hb, 256);
      b.params.push_back(ph.grid);
      b.ptr_params = {{9, want["w"]}};
      to(b, "h");
      partial = std::max(partial, up_to(hb, 256) + f16_partial_bytes(pw, f16_tiles(d, n, pw.tile, false)));
      calls.push_back(std::move(b));
      continue;
    }
    if (wh) to(add("tcb_nll_dh", R, d, n, ph, {z(false, F16_BM), w(false, ph.tile.cols())}), "h");
    if (ww) to(add("tcb_nll_dw", d, n, R, pw, {h(true), z(true, pw.tile.cols())}), "w");
  }
  if (wb && !joined) {
    calls.push_back(make_call("tcb_nll_db", {cdiv(V, 32), 1, 1}, {256, 1, 1}, 0, cat(cat({0, 0, 0, 0}, tail), {0, 0})));
    to(calls.back(), "b");
  }
  Launch l = training_record(node, "linear-nll-grad", nll_source(bool_attr(node, "bias")), std::move(calls),
                             r.end + up_to(partial, 256));
  l.info = {{"rnv", arr({num(R), num(d), num(V)})}, {"pieces", num(pieces)}, {"ctrl_bytes", num(up_to(NLL_CTRL_BYTES, 64))},
            {"path", str("tcgen05-f16x3")}};
  return l;
}

// ---------------------------------------------------------------- headNormRope
static i64 head_rows(i64 D, i64 rotary, i64 v) {
  i64 units = cdiv(rotary / 2, v) + cdiv(D - rotary, 2 * v), lanes = 1;
  while (lanes < std::min<i64>(units, 32)) lanes *= 2;
  return 256 / lanes;
}

static Launch head_launch(const Graph& g, const std::vector<int>& ids) {
  const Node& node = g.nodes[ids[0]];
  const Shape& x = in_shape(g, node, 0);
  const i64 B = x[0], T = x[1], H = x[2], D = x[3], rot = int_attr(node, "rotary");
  const bool back = node.op == "headNormRopeGrad", pairs = bool_attr(node, "interleaved");
  std::map<std::string, int> want;
  for (int i : ids) want[word_attr(g.nodes[i], "wrt")] = i;
  const bool wx = want.count("x"), wg = want.count("gain");
  const bool wide = rot % 8 == 0 && D % 4 == 0;
  const i64 rows = head_rows(D, rot, wide ? 4 : 1);
  i64 heads = 1;
  while (heads * 8 <= H && heads * 2 <= rows) heads *= 2;
  while (heads < H && heads * 2 <= rows && cdiv(T, rows / heads) * B < SM_COUNT * 4) heads *= 2;
  const i64 steps = cdiv(T, rows / heads) * B * cdiv(H, heads);
  const i64 grid = std::min<i64>(steps, SM_COUNT * (back ? 2 : 4));
  i64 flags = (in_shape(g, node, 2).size() == 1 ? 1 : 0) | (bool_attr(node, "headsFirst") ? 2 : 0);
  flags |= (wx ? 4 : 0) | (wg ? 8 : 0);
  const float eps = (float)number_attr(node, "eps");
  uint32_t eps_bits;
  std::memcpy(&eps_bits, &eps, 4);
  const double step = rot ? std::log2(number_attr(node, "base")) / (double)(rot / 2) : 0.0;
  i64 step_bits;
  std::memcpy(&step_bits, &step, 8);
  i64 smem = 0, scratch = 0;
  if (wg) smem = 4 * D * std::max(head_rows(D, rot, 1), wide ? head_rows(D, rot, 4) : 0);
  std::vector<Call> calls;
  calls.push_back(make_call(back ? "tcb_head_norm_rope_grad" : "tcb_head_norm_rope", {grid, 1, 1}, {256, 1, 1}, smem,
                            {B, T, H, flags, heads, (i64)eps_bits, step_bits}));
  if (back && wx && want["x"] != node.id) calls[0].out_node = want["x"];
  if (wg) {
    scratch = grid * D * 4;
    calls.push_back(make_call("tcb_head_gain_finish", {cdiv(D, 8), 1, 1}, {1024, 1, 1}, 0, {grid}));
    if (want["gain"] != node.id) calls[1].out_node = want["gain"];
  }
  std::string code = "// head norm and rotation: heads of " + std::to_string(D) + ", " + std::to_string(rot) + " turned" +
                     (pairs ? " in neighbouring pairs" : "") + "\n#include \"tcb/common.cuh\"\n#define TCB_D " + std::to_string(D) +
                     "\n#define TCB_ROT " + std::to_string(rot) + "\n#define TCB_INTERLEAVED " + (pairs ? "1" : "0") +
                     "\n#include \"tcb/head_norm_rope.cuh\"\n";
  Launch l = training_record(node, back ? "head-norm-rope-grad" : "head-norm-rope", code, std::move(calls), scratch);
  l.info = {{"bthd", arr({num(B), num(T), num(H), num(D)})}, {"heads", num(heads)}};
  return l;
}

// ---------------------------------------------------------------- orthogonalize
static Launch orth_launch(const Graph& g, const Node& node) {
  const Shape& x = in_shape(g, node, 0);
  const i64 m = x[x.size() - 2], n = x[x.size() - 1], batch = size_of(x) / (m * n), steps = int_attr(node, "steps");
  const Value& cv = attr(node, "coeffs");
  const double co[3] = {cv.arr[0].num, cv.arr[1].num, cv.arr[2].num}, eps = number_attr(node, "eps");
  int e[3];
  newton_schulz_scales(node, steps, co, e);
  const bool tall = m > n;
  const i64 s = std::min(m, n), len = std::max(m, n);
  i64 rows = 0, cols = 0;
  if (s <= 64 && len <= 512) rows = 64, cols = 512;
  else if (s <= 128 && len <= 128) rows = 128, cols = 128;
  std::string code = std::string("// Newton-Schulz orthogonalisation") + (rows ? " on one SM" : "") + "\n#include \"tcb/common.cuh\"\n";
  if (rows) code += "#define TCB_ROWS " + std::to_string(rows) + "\n#define TCB_COLS " + std::to_string(cols) + "\n";
  code += "#define TCB_EX " + std::to_string(e[0]) + "\n#define TCB_ES " + std::to_string(e[1]) + "\n#define TCB_EP " +
          std::to_string(e[2]) + "\n#define TCB_NS_A " + f32_literal(co[0]) + "\n#define TCB_NS_B " + f32_literal(co[1]) +
          "\n#define TCB_NS_C " + f32_literal(co[2]) + "\n#define TCB_NS_EPS " + f32_literal(eps) + "\n#include \"tcb/" +
          (rows ? "orth_small" : "orthogonalize") + ".cuh\"\n";
  std::vector<Call> calls;
  if (rows) {
    calls.push_back(make_call("tcb_orth_small", {batch, 1, 1}, {256, 1, 1},
                              (cols / 64 + 2 * (rows / 64)) * (2 * rows * 128) + 16384 + 1024, {m, n, steps}));
    calls[0].err_offset = 0;
    Launch l = training_record(node, "orthogonalize", code, std::move(calls), 256);
    l.info = {{"mn", arr({num(batch), num(m), num(n)})}, {"ctrl_bytes", num(64)}, {"path", str("tcgen05-f16x3")}};
    return l;
  }
  const i64 xp = up_to(n, 8), sp = up_to(s, 8), xplane = 2 * batch * m * xp, splane = 2 * batch * s * sp;
  const i64 parts = std::max<i64>(1, std::min<i64>(NS_PARTS, cdiv(m * n, 4096)));
  Regions r;
  r.add(8 * parts * batch);
  const i64 err = r.add(CTRL_BYTES), x0 = r.add(2 * xplane), x1 = r.add(2 * xplane), s_at = r.add(2 * splane), p_at = r.add(2 * splane);
  const F16Plan gram = f16_plan(s, s, len, batch, NS_CHUNK, true), poly = f16_plan(s, s, s, batch, NS_CHUNK, true),
                app = f16_plan(m, n, s, batch, NS_CHUNK);
  calls.push_back(make_call("tcb_orth_norm", {parts, batch, 1}, {256, 1, 1}, 0, {parts, 0, 0, 0, m, n}));
  calls[0].err_offset = err;
  calls.push_back(make_call("tcb_orth_split", {std::max<i64>(1, std::min<i64>(m * cdiv(n, 1024), SM_COUNT * 8)), batch, 1},
                            {256, 1, 1}, 0, {parts, 0, 0, 0, m, n, x0}));
  auto x_map = [&](i64 off, bool mn, i64 box_rows) { return f16_operand(off, n, m, batch, xp, mn, box_rows); };
  auto s_map = [&](i64 off, i64 box_rows) { return f16_operand(off, s, s, batch, sp, false, box_rows); };
  auto out = [&](i64 off, i64 rs, i64 cs, i64 pitch) {
    return Map{"scratch", off, cs, rs, 2 * batch, pitch * 2, rs * pitch * 2, 32 | F16_FLAG | PAIR_FLAG, 32};
  };
  i64 partial = 0;
  auto add = [&](const std::string& name, i64 M, i64 N, i64 K, const F16Plan& p, std::vector<Map> maps,
                 const std::vector<i64>& params, bool sym) {
    i64 nbytes = 0;
    calls.push_back(f16_gemm(name, M, N, K, batch, p, r.end, std::move(maps), params, err, &nbytes, sym));
    partial = std::max(partial, nbytes);
  };
  const std::string form = tall ? "_tall" : "_wide";
  for (i64 k = 0; k < steps; ++k) {
    const i64 cur = k % 2 ? x1 : x0, nxt = k % 2 ? x0 : x1;
    const std::vector<i64> params = {m, n, cur, nxt, s_at, p_at, k == steps - 1 ? 1 : 0};
    add("tcb_orth_gram" + form, s, s, len, gram, {x_map(cur, tall, F16_BM), x_map(cur, tall, gram.tile.cols()), out(s_at, s, s, sp)}, params, true);
    add("tcb_orth_poly", s, s, s, poly, {s_map(s_at, F16_BM), s_map(s_at, poly.tile.cols()), out(p_at, s, s, sp)}, params, true);
    std::vector<Map> ab = tall ? std::vector<Map>{x_map(cur, false, F16_BM), s_map(p_at, app.tile.cols())}
                               : std::vector<Map>{s_map(p_at, F16_BM), x_map(cur, true, app.tile.cols())};
    ab.push_back(out(nxt, m, n, xp));
    add("tcb_orth_apply" + form, m, n, s, app, std::move(ab), params, false);
  }
  Launch l = training_record(node, "orthogonalize", code, std::move(calls), r.end + up_to(partial, 256));
  l.info = {{"mn", arr({num(batch), num(m), num(n)})}, {"tiles", arr({str(gram.tile.name()), str(poly.tile.name()), str(app.tile.name())})},
            {"ctrl_bytes", num(up_to(CTRL_BYTES, 64))}, {"path", str("tcgen05-f16x3")}};
  return l;
}

// The launch of a training node; false for one that an earlier sibling's launch computes.
static bool training_launch(const Graph& g, const Node& node, const std::map<int, std::vector<int>>& groups, Launch* out) {
  auto it = groups.find(node.id);
  const std::vector<int> ids = it == groups.end() ? std::vector<int>{node.id} : it->second;
  if (ids[0] != node.id) return false;
  for (int i : ids) check_training(g, g.nodes[i]);
  if (node.op == "linearNll") *out = nll_launch(g, ids);
  else if (node.op == "linearNllGrad") *out = nll_grad_launch(g, ids);
  else if (node.op == "orthogonalize") *out = orth_launch(g, node);
  else *out = head_launch(g, ids);
  if (ids.size() > 1) out->nodes = ids;
  std::vector<int> seen;
  i64 n = 0;
  for (int i : out->inputs)
    if (std::find(seen.begin(), seen.end(), i) == seen.end()) {
      seen.push_back(i);
      n += size_of(g.nodes[i].shape);
    }
  for (int i : ids) n += size_of(g.nodes[i].shape);
  out->bytes = 4 * n;
  return true;
}
