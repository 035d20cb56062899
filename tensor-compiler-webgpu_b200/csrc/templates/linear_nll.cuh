// tcb/linear_nll.cuh -- softmax cross entropy of a linear head over a vocabulary, and its gradients,
// without ever holding the logits (the IR ops linearNll and linearNllGrad).
//
//   z = h W + b          h [R, d], W [d, V], b [V]
//   nll_i = log sum_v exp z_iv - z_i,t_i
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t_i]),  dh = dz W^T,  dW = h^T dz,  db = sum_i dz
//
// A row whose target is not one of 0 .. V-1 (a negative one marks padding) is left out: its loss is 0, it
// takes and gives no gradient, and what its row of h holds is never used.
//
// Forward: one matrix product (tcb/gemm_f16x3.cuh) whose epilogue keeps, per row and half tile of columns,
// the running maximum and the sum of exponentials; the last to arrive at 32 rows joins their tiles (a launch of
// its own, tcb_nll_finish, when they are many).  The logits exist in tensor memory and registers only, in units
// of log 2: z2 = log2(e) z is one fma from the sums, its exponential one ex2 (2^-22 relative, as far off as the
// operands' split).
// What the backward needs of it is saved in one opaque value (NllSaved): the scales, b log2(e), each
// row's maximum m and 1 / s of the sum of exponentials below it, and h and W as split for the tensor core, 4 bytes a
// value.  m and s stay two floats: m + log2(s) in one is off by half a step of m, 4e-6 at logits of 100, and so would be
// the gradient of a row whose target is all but certain (and that row's dz would not add up to 0).
// Backward: the vocabulary is walked in pieces (a bounded workspace).  A piece's logits are computed
// again in the forward's order, turned into dz = 2^(z2 - m) g / s - g [v = t] in the epilogue -- as fp16 hi / lo, what the two products after it read;
// |dz| <= |g_i|, so its scale is known before -- and dh += dz W_piece^T and dW_piece = h^T dz follow.
// db's column sums are taken in the dz epilogue, and added up there (or by tcb_nll_db) in the same way.
//
// Range: h, W and dz have one scale each.  A value keeps 22 bits down to 2^-18 of its operand's largest, an absolute
// 2^-39 of the largest below that, and nothing under that.  Results are therefore accurate as float32 in norm; by
// element they are not where small values meet small ones only: dW's column of a class that is improbable in every row
// (dz of 1e-8 of the largest is off by 1e-4 of itself, 1e-12 is lost), dh of a row whose cotangent is as small beside
// the largest, the logits of the other rows beside one row of h with far larger values.
//
// p[] of every kernel: [0..3] the product's (split: [0] blocks of the amax launch; finish: [0] half tiles of a
// row), [4] R, [5] d, [6] V, [7] byte offset of the saved value in scratch (when nobody asks for a backward;
// else the address of the loss), [8..10] byte offsets in it of the row sums, h and W, [11] byte offset in scratch
// of the targets' logits (backward: of the column-sum partials), [12] of the row partials (backward: the piece's
// first column), [13] flags, [14] address of the saved value or 0 (dz: of db or 0).
// in[]: h, W, (b), t forward; t, saved, the loss's cotangent backward.
#pragma once
#include "tcb/gemm_f16x3.cuh"
#include "tcb/nll_common.cuh"

namespace tcb {

// flags: add to dh; join in the product's kernel; no loss; db wanted
constexpr u32 NLL_ADD = 1, NLL_JOIN = 2, NLL_NO_LOSS = 4, NLL_DB = 8;
constexpr u32 NLL_CTRL = F16_CTRL + 512;   // words of the control block: a counter more for each 32 rows or columns joined

// At the start of the saved value; b log2(e) follows at 256 bytes, -inf beyond V up to a multiple of 256.
struct NllScales { float down_h, down_w, z2; };

template <bool BACK> struct Nll {
  const Args& a;
  __device__ __forceinline__ explicit Nll(const Args& args) : a(args) {}
  __device__ __forceinline__ u64 R() const { return (u64)a.p[4]; }
  __device__ __forceinline__ u64 d() const { return (u64)a.p[5]; }
  __device__ __forceinline__ u64 V() const { return (u64)a.p[6]; }
  __device__ __forceinline__ const float* h() const { return reinterpret_cast<const float*>(a.in[0]); }
  __device__ __forceinline__ const float* w() const { return reinterpret_cast<const float*>(a.in[1]); }
  // the row's class, or -1 when it takes no part
  __device__ __forceinline__ int target(u64 row) const {
    return nll_class(ld1(reinterpret_cast<const float*>(a.in[BACK ? 0 : TCB_BIAS ? 3 : 2]) + row), V());
  }
  __device__ __forceinline__ float cotangent(u64 row) const { return ld1(reinterpret_cast<const float*>(a.in[2]) + row); }
  template <class X> __device__ __forceinline__ X* scratch(u64 off) const { return reinterpret_cast<X*>(a.scratch + off); }
  template <class X> __device__ __forceinline__ X* saved(u64 off) const {
    return reinterpret_cast<X*>((BACK ? a.in[1] : a.p[14] ? (u64)a.p[14] : a.scratch + (u64)a.p[7]) + off);
  }
  __device__ __forceinline__ NllScales* scales() const { return saved<NllScales>(0); }
  __device__ __forceinline__ float* bias2() const { return saved<float>(256); }
  __device__ __forceinline__ float2* stats() const { return saved<float2>((u64)a.p[8]); }   // m, 1 / s of every row
  __device__ __forceinline__ float* amax() const { return scratch<float>(0); }
  __device__ __forceinline__ float2* g_scale() const { return scratch<float2>(0); }   // up, down (backward)
};

__device__ __forceinline__ float finite_abs(float x) {
  const float m = fabsf(x);
  return m <= NLL_MAX ? m : 0.0f;   // an infinity or a NaN does not set the scale
}
__device__ __forceinline__ float max4(float m, const float4& q) {
  return fmaxf(fmaxf(m, fmaxf(finite_abs(q.x), finite_abs(q.y))), fmaxf(finite_abs(q.z), finite_abs(q.w)));
}
// the block's maximum of each thread's m (256 threads), in every thread
__device__ __forceinline__ float block_max(float m, float* sh) {
  m = warp_max(m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
  __syncthreads();
  m = sh[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) m = fmaxf(m, sh[k]);
  return m;
}

// Four floats (or fewer at a row's end) of a row of n, from column c.
__device__ __forceinline__ void load4(float (&x)[4], const float* row, u64 c, u64 n, bool wide) {
  if (wide && c + 4 <= n) {
    load<4>(x, row + c);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = c + j < n ? ld1(row + c + j) : 0.0f;
  }
}

// A row-major [rows, n] matrix's hi and lo planes, in blocks of 256 columns (a single block is as wide as n,
// rounded up to 32), zero beyond n up to a multiple of 32.  use(row) false: the row is written as zeros.
template <class F>
__device__ __forceinline__ void split_matrix(const float* x, u32* out, u64 rows, u64 n, float up, u64 block, u64 blocks,
                                             F use) {
  const u64 padded = (n + 31) / 32 * 32, pitch = padded < 256 ? padded : 256;
  const u64 segs = (padded + 1023) / 1024;
  const bool wide = n % 4 == 0 && (reinterpret_cast<u64>(x) & 15) == 0;
  for (u64 u = block; u < rows * segs; u += blocks) {
    const u64 row = u / segs, c = (u % segs) * 1024 + 4 * threadIdx.x;
    if (c >= padded) continue;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (use(row)) load4(v, x + row * n, c, n, wide);
    uint2 hi, lo;
    split2(__fmul_rn(v[0], up), __fmul_rn(v[1], up), hi.x, lo.x);
    split2(__fmul_rn(v[2], up), __fmul_rn(v[3], up), hi.y, lo.y);
    u32* o = out + (((c >> 8) * 2 * rows + row) * pitch + (c & 255)) / 2;
    *reinterpret_cast<uint2*>(o) = hi;
    *reinterpret_cast<uint2*>(o + rows * pitch / 2) = lo;
  }
}

}  // namespace tcb

// The backward has no pass before its first product: a one-off run clears its control block with this (a
// resident program's is its own, and zero between runs).
extern "C" __global__ void __launch_bounds__(128) tcb_gemm_prep(const tcb::Args a) {
  tcb::grid_dependency_sync();
  tcb::f16_clear(a, tcb::NLL_CTRL);
}

// Largest magnitudes of h (rows that take part) and W, a partial pair per block.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_amax(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  f16_clear(a, NLL_CTRL);
  __shared__ float sh[8];
  const Nll<false> n(a);
  const u64 R = n.R(), d = n.d(), V = n.V();
  const int lane = threadIdx.x & 31;
  const u64 warps = (u64)gridDim.x * 8, gw = (u64)blockIdx.x * 8 + (threadIdx.x >> 5);
  float mh = 0.0f, mw = 0.0f;
  const bool wide = d % 4 == 0 && (a.in[0] & 15) == 0;
  for (u64 row = gw; row < R; row += warps) {
    if (n.target(row) < 0) continue;
    for (u64 c = 4 * lane; c < d; c += 128) {
      float x[4];
      load4(x, n.h() + row * d, c, d, wide);
      mh = max4(mh, make_float4(x[0], x[1], x[2], x[3]));
    }
  }
  const u64 total = d * V, T = (u64)gridDim.x * 256, id = (u64)blockIdx.x * 256 + threadIdx.x;
  const u64 quads = (a.in[1] & 15) == 0 ? total / 4 : 0;
  const float4* w4 = reinterpret_cast<const float4*>(n.w());
  u64 i = id;
  for (; i + 7 * T < quads; i += 8 * T) {   // eight loads in flight
    float4 q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = __ldg(w4 + i + k * T);
#pragma unroll
    for (int k = 0; k < 8; ++k) mw = max4(mw, q[k]);
  }
  for (; i < quads; i += T) mw = max4(mw, __ldg(w4 + i));
  for (i = 4 * quads + id; i < total; i += T) mw = fmaxf(mw, finite_abs(ld1(n.w() + i)));
  mh = block_max(mh, sh);
  mw = block_max(mw, sh);
  if (threadIdx.x == 0) {
    n.amax()[2 * blockIdx.x] = mh;
    n.amax()[2 * blockIdx.x + 1] = mw;
  }
}

// The scales from the partial maxima (every block for itself; block 0 writes them down), then b log2(e), h
// and W split.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_split(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float sh[8];
  const Nll<false> n(a);
  float mh = 0.0f, mw = 0.0f;
  for (u32 i = threadIdx.x; i < (u32)a.p[0]; i += 256) {
    const float2 m = reinterpret_cast<const float2*>(n.amax())[i];
    mh = fmaxf(mh, m.x);
    mw = fmaxf(mw, m.y);
  }
  const int kh = scale_exponent(block_max(mh, sh)), kw = scale_exponent(block_max(mw, sh));
  if (blockIdx.x == 0 && threadIdx.x == 0)   // the clamp: an accumulator of 0 times inf would be NaN
    *n.scales() = NllScales{pow2(-kh), pow2(-kw), fminf(pow2(-kh) * pow2(-kw) * NLL_LOG2E, NLL_MAX)};
  const u64 V = n.V(), padded = (V + 255) / 256 * 256;
  for (u64 v = (u64)blockIdx.x * 256 + threadIdx.x; v < padded; v += (u64)gridDim.x * 256) {
    const float b = TCB_BIAS && v < V ? ld1(reinterpret_cast<const float*>(a.in[2]) + v) : 0.0f;
    n.bias2()[v] = v < V ? nll_bias2(b) : TCB_MINUS_INF;
  }
  // the last blocks take h, about its share of the pieces of rows (of the values, W's 600 rows of 3 fell to one
  // block: 203 us)
  const u64 hv = n.R() * ((n.d() + 1023) / 1024), wv = n.d() * ((V + 1023) / 1024);
  u64 hb = gridDim.x * hv / (hv + wv);
  hb = hb < 1 ? 1 : hb > gridDim.x - 1 ? gridDim.x - 1 : hb;
  const u64 wb = gridDim.x - hb;
  if (blockIdx.x < wb)
    split_matrix(n.w(), n.saved<u32>((u64)a.p[10]), n.d(), V, pow2(kw), blockIdx.x, wb, [](u64) { return true; });
  else
    split_matrix(n.h(), n.saved<u32>((u64)a.p[9]), n.R(), n.d(), pow2(kh), blockIdx.x - wb, hb,
                 [&](u64 row) { return n.target(row) >= 0; });
}

namespace tcb {

// The 32 scaled logits of a block from their sums and the bias, a column a lane (loaded a block ahead), which
// the warp's shared memory hands to every lane.
__device__ __forceinline__ void nll_logits(const F16Epi& e, float (&v)[32], float z2, float bias) {
  __syncwarp();
  e.vec[e.lane] = bias;
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const float4 b = *reinterpret_cast<const float4*>(e.vec + 4 * c);
    fma2(v[4 * c], v[4 * c + 1], z2, z2, b.x, b.y);
    fma2(v[4 * c + 2], v[4 * c + 3], z2, z2, b.z, b.w);
  }
}
// This lane's column of the block at c0 of a tile, the last one again beyond N.
__device__ __forceinline__ u32 nll_column(const F16Epi& e, int c0) {
  const u32 col = (u32)(e.T.n0 + c0 + e.lane), last = (e.N + 31) / 32 * 32 - 1;
  return col < last ? col : last;
}
// The target's place among 32 columns as a bit: comparing an index with each would be turned into an
// indexed read and keep the sums in local memory.
__device__ __forceinline__ u32 nll_bit(int t, u32 col) {
  return t >= (int)col && t < (int)col + 32 ? 1u << (t - (int)col) : 0u;
}

// A warp's arrival at one of n: true, in all lanes, for the last, which leaves the counter at zero.
__device__ __forceinline__ bool nll_last(const Args& a, u32 counter, u32 n, int lane) {
  __threadfence();
  __syncwarp();
  u32* c = reinterpret_cast<u32*>(a.p[15]) + 4 + 8 * 2 * 148 + counter;   // behind the divided tiles' counters
  u32 old = 0;
  if (lane == 0) old = atomicAdd(c, 1u);
  const bool last = __shfl_sync(0xffffffffu, old, 0) == n - 1;
  if (last) {
    if (lane == 0) *c = 0u;
    __threadfence();
  }
  return last;
}
// Half tiles k, k + step, ... of a row joined, eight loads in flight.
__device__ __forceinline__ void nll_join_tiles(const float2* part, u64 R, u64 row, u32 k, u32 step, u32 tiles, float& m,
                                               float& s) {
  m = TCB_MINUS_INF;
  s = 0.0f;
  for (; k + 7 * step < tiles; k += 8 * step) {
    float2 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __ldcg(part + (u64)(k + i * step) * R + row);
#pragma unroll
    for (int i = 0; i < 8; ++i) nll_join(m, s, x[i]);
  }
  for (; k < tiles; k += step) nll_join(m, s, __ldcg(part + (u64)k * R + row));
}
__device__ __forceinline__ void nll_write(const Nll<false>& n, u64 row, float m, float s) {
  const Args& a = n.a;
  if (!((u32)a.p[13] & NLL_NO_LOSS))
    reinterpret_cast<float*>(a.p[14] ? (u64)a.p[7] : a.out)[row] =
        nll_loss(m, s, __ldcg(n.scratch<float>((u64)a.p[11]) + row), n.target(row), reinterpret_cast<const float*>(a.in[2]));
  n.stats()[row] = make_float2(m, 1.0f / s);
}

// Forward epilogue: a row's maximum and sum of exponentials over the half tile's columns, the target's
// logit.  Columns of -inf (a masked part of the vocabulary, the padding) leave the sum alone.
template <int BN>
struct NllForward {
  const Args& a;
  const float* bias2;
  float z2, m, s, bias;
  int t;
  __device__ __forceinline__ explicit NllForward(const Args& args) : a(args) {}
  __device__ __forceinline__ void start(unsigned char*) {
    const Nll<false> n(a);
    z2 = n.scales()->z2;
    bias2 = n.bias2();
  }
  __device__ __forceinline__ void begin(const F16Epi& e) {
    const Nll<false> n(a);
    m = TCB_MINUS_INF;
    s = 0.0f;
    t = e.row < n.R() ? n.target(e.row) : -1;
    bias = bias2[nll_column(e, e.c0)];
  }
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    const u32 col = (u32)(e.T.n0 + c0);
    nll_logits(e, v, z2, bias);
    bias = bias2[nll_column(e, c0 + 32)];
    float mx = m;
#pragma unroll
    for (int j = 0; j < 32; ++j) mx = fmaxf(mx, v[j]);
    const u32 mine = nll_bit(t, col);
    if (mine) {
      float z = 0.0f;
#pragma unroll
      for (int j = 0; j < 32; ++j) z = (mine >> j) & 1 ? v[j] : z;
      Nll<false>(a).template scratch<float>((u64)a.p[11])[e.row] = z;
    }
    const float safe = mx == TCB_MINUS_INF ? 0.0f : mx;
    float q[4] = {s * ex2(m - safe), 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      add2(v[j], v[j + 1], -safe, -safe);
      add2(q[j & 3], q[(j & 3) + 1], ex2(v[j]), ex2(v[j + 1]));
    }
    s = (q[0] + q[1]) + (q[2] + q[3]);
    m = mx;
  }
  __device__ __forceinline__ void end(const F16Epi& e) {
    const Nll<false> n(a);
    float2* part = n.template scratch<float2>((u64)a.p[12]);
    if (e.row < n.R()) part[(u64)(e.T.n0 + e.c0) / (BN / 2) * n.R() + e.row] = make_float2(m, s);
    if (!((u32)a.p[13] & NLL_JOIN)) return;
    const u32 halves = ((u32)n.V() + BN / 2 - 1) / (BN / 2);
    if (!nll_last(a, (u32)e.T.m0 / 32 + e.q, halves, e.lane) || e.row >= n.R()) return;
    nll_join_tiles(part, n.R(), e.row, 0, 1, halves, m, s);
    nll_write(n, e.row, m, s);
  }
  __device__ __forceinline__ void done(const F16Epi&) {}
};

// Backward epilogue: logits to dz, split for the products that read it; its column sums for db.
template <int BN>
struct NllDz {
  const Args& a;
  const TmaDesc* map;
  const float* bias2;
  float* part_row;   // where this lane's column sums go
  float z2, up, down, m, g, p, bias;   // p: what an exponential is multiplied by
  int t;
  __device__ __forceinline__ explicit NllDz(const GemmParams& P) : a(P.a), map(&P.maps[2]) {}
  // The cotangent's scale: each CTA's epilogue warps look through all of it behind the first product.
  __device__ __forceinline__ void start(unsigned char* smem) {
    const Nll<true> n(a);
    z2 = n.scales()->z2;
    bias2 = n.bias2() + (u64)a.p[12];
    float m = 0.0f;
    for (u64 i = threadIdx.x - 128; i < n.R(); i += 8 * 256) {   // sixteen loads in flight
      float x[8];
      int c[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const u64 r = i + 256 * k < n.R() ? i + 256 * k : i;   // (a branch would have the loads wait one for another)
        x[k] = n.cotangent(r);
        c[k] = n.target(r);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, c[k] >= 0 ? finite_abs(x[k]) : 0.0f);
    }
    m = warp_max(m);
    float* sh = reinterpret_cast<float*>(smem);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x / 32 - 4] = m;
    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, sh[k]);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const int k = scale_exponent(m);
    up = pow2(k);
    down = pow2(-k);
    if (blockIdx.x == 0 && threadIdx.x == 128) *n.g_scale() = make_float2(up, down);
  }
  __device__ __forceinline__ void begin(const F16Epi& e) {
    const Nll<true> n(a);
    const u64 row = e.row < n.R() ? e.row : n.R() - 1;
    t = n.target(row);
    const float2 stats = n.stats()[row];
    m = stats.x;
    g = n.cotangent(row) * up;
    p = g * stats.y;
    if (e.row != row) t = -1;
    part_row = n.template scratch<float>((u64)a.p[11]) + ((u64)e.T.m0 / 32 + e.q) * n.V() + (u64)a.p[12] + e.lane;
    bias = bias2[nll_column(e, e.c0)];
  }
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    const Nll<true> n(a);
    const u32 pc = (u32)(e.T.n0 + c0), col = (u32)a.p[12] + pc;
    nll_logits(e, v, z2, bias);
    bias = bias2[nll_column(e, c0 + 32)];
    const u32 mine = nll_bit(t, col);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      add2(v[j], v[j + 1], -m, -m);
      v[j] = ex2(v[j]);
      v[j + 1] = ex2(v[j + 1]);
    }
#pragma unroll
    for (int j = 0; j < 32; j += 2) mul2(v[j], v[j + 1], p, p);
    if (__any_sync(0xffffffffu, mine != 0u)) {   // in one block of 8 at 8192 classes
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = (mine >> j) & 1 ? v[j] - g : v[j];
    }
    if (t < 0) {   // not by g = 0: an excluded row's logits may be anything
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0.0f;
    }
    stage_split32(e, v);
    const bool db = ((u32)a.p[13] & NLL_DB) != 0;
    const float sum = db ? column_sums32(v, e.lane) : 0.0f;   // while the values are on their way to shared memory
    send_split32(e, map, (int)(pc & 255), e.T.m0 + 32 * e.q, (int)(pc >> 8));
    const bool in = pc + e.lane < e.N;
    if (db && in) part_row[pc] = sum * down;
    if (!((u32)a.p[13] & NLL_JOIN)) return;
    const float* part = n.template scratch<float>((u64)a.p[11]) + col + e.lane;
    const u32 rows = ((u32)n.R() + 31) / 32;
    if (!nll_last(a, col / 32, rows, e.lane) || !in) return;
    float x = 0.0f;
#pragma unroll 8
    for (u32 k = 0; k < rows; ++k) x += __ldcg(part + (u64)k * n.V());
    reinterpret_cast<float*>(a.p[14])[col + e.lane] = x;
  }
  __device__ __forceinline__ void end(const F16Epi&) {}
  __device__ __forceinline__ void done(const F16Epi& e) {
    if (e.lane == 0) bulk_wait_all();
  }
};

// dh (rows of d, added to over the pieces) or dW (rows of V, from the piece's first column), scaled back.
template <bool DW>
struct NllOut {
  const Args& a;
  float* out;
  float x, y;
  __device__ static int exponent(float power) { return (int)(__float_as_uint(power) >> 23) - 127; }
  __device__ __forceinline__ NllOut(const Args& args, u64 o) : a(args), out(reinterpret_cast<float*>(o)) {}
  __device__ __forceinline__ void start(unsigned char*) {
    const Nll<true> n(a);
    // the two powers of two as two of about one size: operands far from 1 would leave the range half way
    const int k = exponent(DW ? n.scales()->down_h : n.scales()->down_w) + exponent(n.g_scale()->y);
    x = pow2(k >> 1);
    y = pow2(k - (k >> 1));
  }
  __device__ __forceinline__ void begin(const F16Epi&) {}
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    turn32(e, v);
    const u32 col = (u32)(e.T.n0 + c0) + e.lane;
    if (col >= e.N) return;
    const u64 ld = DW ? (u64)a.p[6] : (u64)a.p[5];
    const u32 row0 = (u32)e.T.m0 + 32 * e.q;
    float* o = out + row0 * ld + (DW ? (u64)a.p[12] : 0) + col;
    const int rows = (int)(e.M - row0 < 32 ? e.M - row0 : 32);
#pragma unroll
    for (int r = 0; r < 32; ++r) v[r] = v[r] * x * y;
    if (!DW && ((u32)a.p[13] & NLL_ADD)) {
#pragma unroll
      for (int r = 0; r < 32; ++r)
        if (r < rows) v[r] += o[(u64)r * ld];
    }
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (r < rows) o[(u64)r * ld] = v[r];
  }
  __device__ __forceinline__ void end(const F16Epi&) {}
  __device__ __forceinline__ void done(const F16Epi&) {}
};

}  // namespace tcb

#define TCB_NLL_GEMM(NAME, TILE, BN, CTAS, AMN, BMN, EPI, ...)                                                      \
  extern "C" __global__ void TCB_F16_CLUSTER_##CTAS __launch_bounds__(tcb::HG_THREADS, 1)                           \
      NAME##_##TILE(const __grid_constant__ tcb::GemmParams P) {                                                    \
    tcb::EPI epi(__VA_ARGS__);                                                                                      \
    tcb::gemm_f16x3<BN, CTAS, AMN, BMN, false, true, 256>(tcb::f16_job(P), reinterpret_cast<u32*>(P.a.p[15]), epi); \
  }
// logits and dz: h K-major, W MN-major (its rows run along the vocabulary); dh: dz and W K-major (along the
// vocabulary); dW: h^T and dz, both MN-major (along d and along the vocabulary)
#define TCB_NLL_GEMMS(TILE, BN, CTAS)                                                 \
  TCB_NLL_GEMM(tcb_nll_logits, TILE, BN, CTAS, false, true, NllForward<BN>, P.a)      \
  TCB_NLL_GEMM(tcb_nll_dz, TILE, BN, CTAS, false, true, NllDz<BN>, P)                 \
  TCB_NLL_GEMM(tcb_nll_dh, TILE, BN, CTAS, false, false, NllOut<false>, P.a, P.a.out) \
  TCB_NLL_GEMM(tcb_nll_dw, TILE, BN, CTAS, true, true, NllOut<true>, P.a, P.a.out)
TCB_F16_TILES(TCB_NLL_GEMMS)

// dh and dW in one launch where their CTAs find room side by side: the first p[14] CTAs are dh's, maps 2 and 3,
// p[7] (plan), p[8] (partial sums) and p[9] (address) dW's.
template <int BH, int BW>
__device__ __forceinline__ void nll_both(const tcb::GemmParams& P) {
  using namespace tcb;
  const Args& a = P.a;
  u32* err = reinterpret_cast<u32*>(a.p[15]);
  F16Job j = f16_job(P);
  if (blockIdx.x < (u32)a.p[14]) {
    j.grid = (u32)a.p[14];
    NllOut<false> epi(a, a.out);
    gemm_f16x3<BH, 1, false, false, false, true, 256>(j, err, epi);
  } else {
    j = F16Job{&P.maps[2], &P.maps[3], (u32)a.p[5], j.K, j.M, 1, (u32)a.p[7], (u32)((u64)a.p[7] >> 32),
               blockIdx.x - (u32)a.p[14], gridDim.x - (u32)a.p[14], reinterpret_cast<float*>(a.scratch + (u64)a.p[8]),
               j.counters + 8 * 148};
    NllOut<true> epi(a, (u64)a.p[9]);
    gemm_f16x3<BW, 1, true, true, false, true, 256>(j, err, epi);
  }
}
#define TCB_NLL_BOTH(BH, BW)                                                                                          \
  extern "C" __global__ void __launch_bounds__(tcb::HG_THREADS, 1)                                                    \
      tcb_nll_both_##BH##_##BW(const __grid_constant__ tcb::GemmParams P) { nll_both<BH, BW>(P); }
TCB_NLL_BOTH(64, 64)
TCB_NLL_BOTH(64, 128)
TCB_NLL_BOTH(128, 64)
TCB_NLL_BOTH(128, 128)

// Joins a row's tiles: a block of 8 warps takes 32 rows, warp k the half tiles k, k + 8, ...
extern "C" __global__ void __launch_bounds__(256) tcb_nll_finish(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float2 sh[8][32];
  const Nll<false> n(a);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const u64 R = n.R(), row = (u64)blockIdx.x * 32 + lane;
  float m = TCB_MINUS_INF, s = 0.0f;
  if (row < R) nll_join_tiles(n.scratch<float2>((u64)a.p[12]), R, row, w, 8, (u32)a.p[0], m, s);
  sh[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w == 0 && row < R) {
    for (int k = 1; k < 8; ++k) nll_join(m, s, sh[k][lane]);
    nll_write(n, row, m, s);
  }
}

// db: the partial column sums (one per 32 rows) added up, 32 columns a block.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_db(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float sh[8][32];
  const Nll<true> n(a);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const u64 V = n.V(), parts = (n.R() + 31) / 32, col = (u64)blockIdx.x * 32 + lane;
  const float* p = n.scratch<float>((u64)a.p[11]);
  float s = 0.0f;
  if (col < V) {
#pragma unroll 4
    for (u64 k = w; k < parts; k += 8) s += p[k * V + col];
  }
  sh[w][lane] = s;
  __syncthreads();
  if (w == 0 && col < V) {
    for (int k = 1; k < 8; ++k) s += sh[k][lane];
    reinterpret_cast<float*>(a.out)[col] = s;
  }
}
