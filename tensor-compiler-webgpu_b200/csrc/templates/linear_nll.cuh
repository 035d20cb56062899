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
// Forward: one matrix product (tcb/gemm_f16x3.cuh) whose epilogue keeps, per row and half tile of columns, the
// running maximum and the sum of exponentials; tcb_nll_finish joins a row's tiles.  The logits exist in
// tensor memory only.
// Backward: the vocabulary is walked in pieces of TCB's host's choosing (a bounded workspace).  A piece's
// logits are computed again, turned into dz in the epilogue -- as fp16 hi / lo, what the two products
// after it read; |dz| <= |g_i|, so its scale is known before -- and dh += dz W_piece^T and
// dW_piece = h^T dz follow.  db's column sums are taken in the dz epilogue.  lse_i is nll_i + z_i,t_i,
// with the target's logit as a dot product in double, so the forward hands over no more than its loss.
//
// dz below 2^-40 of the largest |g_i| rounds to zero, and keeps fewer than 22 bits below 2^-18 of it: the
// gradient of a class whose probability is that small in every row has that absolute accuracy, which is
// beneath the float32 rounding of the sums it enters.
//
// p[] of every kernel: [0..3] the product's M, N, K, batch (amax / split / finish: [0] the blocks of the
// amax launch), [4] R, [5] d, [6] V, [7..11] byte offsets in scratch of h's split, W's split, the row
// statistics, dz, the column-sum partials, [12] first column of the piece, [13] flags.
// in[]: h, W, (b), t, then in the backward nll and the loss's cotangent.
#pragma once
#include "tcb/gemm_f16x3.cuh"

#ifndef TCB_BIAS
#define TCB_BIAS 1
#endif

namespace tcb {

constexpr int NLL_T = TCB_BIAS ? 3 : 2;
constexpr u32 NLL_BACKWARD = 1, NLL_ADD = 2;

struct NllScales { float up_h, up_w, up_g, down_h, down_w, down_g; };   // at the start of scratch

struct Nll {
  const Args& a;
  __device__ explicit Nll(const Args& args) : a(args) {}
  __device__ u64 R() const { return (u64)a.p[4]; }
  __device__ u64 d() const { return (u64)a.p[5]; }
  __device__ u64 V() const { return (u64)a.p[6]; }
  __device__ const float* h() const { return reinterpret_cast<const float*>(a.in[0]); }
  __device__ const float* w() const { return reinterpret_cast<const float*>(a.in[1]); }
  __device__ float bias(u64 v) const { return TCB_BIAS ? ld1(reinterpret_cast<const float*>(a.in[2]) + v) : 0.0f; }
  // the row's class, or -1 when it takes no part
  __device__ int target(u64 row) const {
    const float t = ld1(reinterpret_cast<const float*>(a.in[NLL_T]) + row);
    return t >= 0.0f && t < (float)V() ? (int)t : -1;
  }
  template <class X> __device__ X* at(u64 off) const { return reinterpret_cast<X*>(a.scratch + off); }
  __device__ NllScales* scales() const { return at<NllScales>(0); }
  __device__ float* amax() const { return at<float>(512); }
  __device__ u32* h_split() const { return at<u32>((u64)a.p[7]); }
  __device__ u32* w_split() const { return at<u32>((u64)a.p[8]); }
};

__device__ __forceinline__ float finite_abs(float x) {
  const float m = fabsf(x);
  return m <= 3.402823466e38f ? m : 0.0f;   // an infinity or a NaN does not set the scale
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

// A row-major [rows, n] matrix's hi and lo planes, row pitch n rounded up to 8 (the values between n and
// the pitch are never read).  use(row) false: the row is written as zeros.
template <class F>
__device__ __forceinline__ void split_matrix(const float* x, u32* out, u64 rows, u64 n, float up, u64 block, u64 blocks,
                                             F use) {
  const u64 pitch = (n + 7) / 8 * 8, plane = rows * pitch / 2;
  const u64 segs = (n + 1023) / 1024;
  const bool wide = n % 4 == 0 && (reinterpret_cast<u64>(x) & 15) == 0;
  for (u64 u = block; u < rows * segs; u += blocks) {
    const u64 row = u / segs, c = (u % segs) * 1024 + 4 * threadIdx.x;
    if (c >= n) continue;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (use(row)) load4(v, x + row * n, c, n, wide);
    uint2 hi, lo;
    split2(__fmul_rn(v[0], up), __fmul_rn(v[1], up), hi.x, lo.x);
    split2(__fmul_rn(v[2], up), __fmul_rn(v[3], up), hi.y, lo.y);
    u32* o = out + (row * pitch + c) / 2;
    *reinterpret_cast<uint2*>(o) = hi;
    *reinterpret_cast<uint2*>(o + plane) = lo;
  }
}

}  // namespace tcb

// Largest magnitudes of h (rows that take part), W and, in the backward, the cotangent, a partial per
// block; the backward's row statistics {lse, g, target} too.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_amax(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.p[15]) *reinterpret_cast<u32*>(a.p[15]) = 0u;
  __shared__ float sh[8];
  const Nll n(a);
  const u64 R = n.R(), d = n.d(), V = n.V();
  const bool backward = ((u32)a.p[13] & NLL_BACKWARD) != 0;
  const int lane = threadIdx.x & 31;
  const u64 warps = (u64)gridDim.x * 8, gw = (u64)blockIdx.x * 8 + (threadIdx.x >> 5);
  float mh = 0.0f, mw = 0.0f, mg = 0.0f;
  const bool wide = d % 4 == 0 && (a.in[0] & 15) == 0;
  for (u64 row = gw; row < R; row += warps) {
    const int t = n.target(row);
    if (t >= 0)
      for (u64 c = 4 * lane; c < d; c += 128) {
        float x[4];
        load4(x, n.h() + row * d, c, d, wide);
        mh = max4(mh, make_float4(x[0], x[1], x[2], x[3]));
      }
    if (backward) {
      float lse = 0.0f, g = 0.0f;
      if (t >= 0) {
        g = ld1(reinterpret_cast<const float*>(a.in[NLL_T + 2]) + row);
        mg = fmaxf(mg, finite_abs(g));
        double z = 0.0;
        for (u64 k = lane; k < d; k += 32) z += (double)ld1(n.h() + row * d + k) * (double)ld1(n.w() + k * V + (u64)t);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        lse = (float)(z + (double)n.bias((u64)t) + (double)ld1(reinterpret_cast<const float*>(a.in[NLL_T + 1]) + row));
      }
      if (lane == 0) n.at<float4>((u64)a.p[9])[row] = make_float4(lse, g, __int_as_float(t), 0.0f);
    }
  }
  const u64 total = d * V, T = (u64)gridDim.x * 256, id = (u64)blockIdx.x * 256 + threadIdx.x;
  const u64 quads = (a.in[1] & 15) == 0 ? total / 4 : 0;
  const float4* w4 = reinterpret_cast<const float4*>(n.w());
#pragma unroll 4
  for (u64 i = id; i < quads; i += T) mw = max4(mw, __ldg(w4 + i));
  for (u64 i = 4 * quads + id; i < total; i += T) mw = fmaxf(mw, finite_abs(ld1(n.w() + i)));
  mh = block_max(mh, sh);
  mw = block_max(mw, sh);
  mg = block_max(mg, sh);
  if (threadIdx.x == 0) {
    float* m = n.amax() + 3 * blockIdx.x;
    m[0] = mh; m[1] = mw; m[2] = mg;
  }
}

// The scales from the partial maxima (every block for itself; block 0 writes them down), then h and W split.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_split(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float sh[8];
  const Nll n(a);
  float mh = 0.0f, mw = 0.0f, mg = 0.0f;
  for (u32 i = threadIdx.x; i < (u32)a.p[0]; i += 256) {
    const float* m = n.amax() + 3 * i;
    mh = fmaxf(mh, m[0]); mw = fmaxf(mw, m[1]); mg = fmaxf(mg, m[2]);
  }
  const int kh = scale_exponent(block_max(mh, sh)), kw = scale_exponent(block_max(mw, sh));
  const int kg = scale_exponent(block_max(mg, sh));
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *n.scales() = NllScales{pow2(kh), pow2(kw), pow2(kg), pow2(-kh), pow2(-kw), pow2(-kg)};
  // the last blocks take h, about its share of the values
  const u64 hv = n.R() * n.d(), wv = n.d() * n.V();
  u64 hb = gridDim.x * hv / (hv + wv);
  hb = hb < 1 ? 1 : hb > gridDim.x - 1 ? gridDim.x - 1 : hb;
  const u64 wb = gridDim.x - hb;
  if (blockIdx.x < wb)
    split_matrix(n.w(), n.w_split(), n.d(), n.V(), pow2(kw), blockIdx.x, wb, [](u64) { return true; });
  else
    split_matrix(n.h(), n.h_split(), n.R(), n.d(), pow2(kh), blockIdx.x - wb, hb,
                 [&](u64 row) { return n.target(row) >= 0; });
}

namespace tcb {

// Forward epilogue: a row's maximum and sum of exponentials over the tile's columns, the target's logit.
// A block of -inf logits (a masked part of the vocabulary) leaves the sum alone.
template <int BN>
struct NllForward {
  const Args& a;
  float dh, dw, m, s;
  int t;
  __device__ explicit NllForward(const Args& args) : a(args) {}
  __device__ __forceinline__ void begin(const F16Epi& e) {
    const Nll n(a);
    dh = n.scales()->down_h;
    dw = n.scales()->down_w;
    m = bits(0xff800000u);
    s = 0.0f;
    t = e.row < n.R() ? n.target(e.row) : -1;
  }
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    const Nll n(a);
    const u32 col = (u32)(e.T.n0 + c0);
    const int left = (int)((u32)n.V() - col);   // > 0
    float mx = m;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = j < left ? v[j] * dh * dw + n.bias(col + (j < left ? j : 0)) : bits(0xff800000u);
      mx = fmaxf(mx, v[j]);
    }
    // a bit per column, not an index compared: the compiler would turn that into an indexed read of v and
    // keep the sums in local memory
    const u32 mine = t >= (int)col && t < (int)col + 32 ? 1u << (t - (int)col) : 0u;
    if (mine) {
      float z = 0.0f;
#pragma unroll
      for (int j = 0; j < 32; ++j) z = (mine >> j) & 1 ? v[j] : z;
      n.at<float>((u64)a.p[9])[e.row] = z;
    }
    const float safe = mx == bits(0xff800000u) ? 0.0f : mx;
    float q[4] = {s * expf(m - safe), 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 32; ++j) q[j & 3] += expf(v[j] - safe);
    s = (q[0] + q[1]) + (q[2] + q[3]);
    m = mx;
  }
  __device__ __forceinline__ void end(const F16Epi& e) {
    const Nll n(a);
    if (e.row < n.R()) n.at<float2>((u64)a.p[10])[(u64)(e.T.n0 + e.c0) / (BN / 2) * n.R() + e.row] = make_float2(m, s);
  }
  __device__ __forceinline__ void done(const F16Epi&) {}
};

// Backward epilogue: logits to dz, split for the products that read it; its column sums for db.
struct NllDz {
  const Args& a;
  const TmaDesc* map;
  float dh, dw, ug, lse, g;
  int t;
  __device__ NllDz(const GemmParams& P) : a(P.a), map(&P.maps[4]) {}
  __device__ __forceinline__ void begin(const F16Epi& e) {
    const Nll n(a);
    dh = n.scales()->down_h;
    dw = n.scales()->down_w;
    ug = n.scales()->up_g;
    const float4 s = e.row < n.R() ? n.at<float4>((u64)a.p[9])[e.row]
                                   : make_float4(0.0f, 0.0f, __int_as_float(-1), 0.0f);
    lse = s.x;
    g = s.y;
    t = __float_as_int(s.z);
  }
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    const Nll n(a);
    const u32 pc = (u32)(e.T.n0 + c0), col = (u32)a.p[12] + pc;
    const int left = (int)((u32)a.p[1] - pc);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float z = v[j] * dh * dw + n.bias(col + (j < left ? j : 0));
      float p = expf(z - lse);
      if (t - (int)col == j) p -= 1.0f;
      v[j] = t >= 0 && j < left ? g * p : 0.0f;
    }
    float c[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) c[j] = v[j];
    const float sum = column_sums32(c, e.lane);
    if (e.lane < left)
      n.at<float>((u64)a.p[11])[((u64)e.T.m0 / 32 + e.q) * n.V() + col + e.lane] = sum;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= ug;
    store_split32(e, map, v, (int)pc, e.T.m0 + 32 * e.q, 0, 1);
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
  float x, y;
  __device__ explicit NllOut(const Args& args) : a(args) {}
  __device__ __forceinline__ void begin(const F16Epi&) {
    const NllScales* s = Nll(a).scales();
    x = DW ? s->down_h : s->down_w;
    y = s->down_g;
  }
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    turn32(e, v);
    const u32 col = (u32)(e.T.n0 + c0) + e.lane;
    if (col >= (u32)a.p[1]) return;
    const u64 ld = DW ? (u64)a.p[6] : (u64)a.p[5];
    const u64 row0 = (u64)e.T.m0 + 32 * e.q;
    float* o = reinterpret_cast<float*>(a.out) + row0 * ld + (DW ? (u64)a.p[12] : 0) + col;
    const int rows = (int)((u64)a.p[0] - row0 < 32 ? (u64)a.p[0] - row0 : 32);
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

#define TCB_NLL_GEMM(NAME, BN, AMN, BMN, EPI, ARG)                                                                    \
  extern "C" __global__ void __launch_bounds__(tcb::HG_THREADS, 1) NAME##_##BN(const __grid_constant__ tcb::GemmParams P) { \
    tcb::EPI epi(ARG);                                                                                                \
    tcb::gemm_f16x3<BN, AMN, BMN, false, 256>(P, epi);                                                                \
  }
// logits and dz: h K-major, W MN-major (its rows run along the vocabulary); dh: dz and W K-major (along the
// vocabulary); dW: h^T and dz, both MN-major (along d and along the vocabulary)
#define TCB_NLL_GEMMS(BN)                                          \
  TCB_NLL_GEMM(tcb_nll_logits, BN, false, true, NllForward<BN>, P.a) \
  TCB_NLL_GEMM(tcb_nll_dz, BN, false, true, NllDz, P)              \
  TCB_NLL_GEMM(tcb_nll_dh, BN, false, false, NllOut<false>, P.a)   \
  TCB_NLL_GEMM(tcb_nll_dw, BN, true, true, NllOut<true>, P.a)
TCB_NLL_GEMMS(256)
TCB_NLL_GEMMS(128)
TCB_NLL_GEMMS(64)

// Joins a row's tiles: a block of 8 warps takes 32 rows, warp k the tiles k, k + 8, ...
extern "C" __global__ void __launch_bounds__(256) tcb_nll_finish(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float2 sh[8][32];
  const Nll n(a);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const u64 R = n.R(), row = (u64)blockIdx.x * 32 + lane;
  const u32 tiles = (u32)a.p[0];
  const float2* part = n.at<float2>((u64)a.p[10]);
  float m = bits(0xff800000u), s = 0.0f;
  auto join = [&](const float2& x) {
    const float mx = fmaxf(m, x.x), safe = mx == bits(0xff800000u) ? 0.0f : mx;
    s = s * expf(m - safe) + x.y * expf(x.x - safe);
    m = mx;
  };
  if (row < R) {
#pragma unroll 4
    for (u32 k = w; k < tiles; k += 8) join(part[(u64)k * R + row]);
  }
  sh[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w == 0 && row < R) {
    for (int k = 1; k < 8; ++k) join(sh[k][lane]);
    reinterpret_cast<float*>(a.out)[row] =
        n.target(row) >= 0 ? (m - n.at<float>((u64)a.p[9])[row]) + logf(s) : 0.0f;
  }
}

// db: the partial column sums (one per 32 rows) added up, 32 columns a block.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_db(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float sh[8][32];
  const Nll n(a);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const u64 V = n.V(), parts = (n.R() + 31) / 32, col = (u64)blockIdx.x * 32 + lane;
  const float* p = n.at<float>((u64)a.p[11]);
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
