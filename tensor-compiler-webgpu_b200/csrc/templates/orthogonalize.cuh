// tcb/orthogonalize.cuh -- Newton-Schulz orthogonalisation of a matrix, or of each of a stack (the IR op
// orthogonalize: the update of the Muon optimiser).
//
//   X = G / (|G|_F + eps), then TCB_NS_STEPS times, on the short side of G:
//   wide (m <= n):  S = X X^T,  P = b S + c S S,  X = a X + P X
//   tall (m > n):   S = X^T X,  P = b S + c S S,  X = a X + X P
//
// Three products a step (tcb/gemm_f16x3.cuh), and nothing between them: S, P and X exist only as the fp16
// hi / lo pairs that the next product reads, written by the epilogue of the one before (22 bits of each
// value, its rounding below the float32 sum it came from).  Their scales are fixed: |X|_F = 1 bounds the
// singular values of every step, so the host knows the largest entry X, S and P can have (2^TCB_EX,
// 2^TCB_ES and 2^TCB_EP scale them into fp16).  S and P are symmetric: half of their tiles are computed,
// the rest mirrored.  A tall matrix is never transposed: the tensor core reads X along either side.
// Chains of 128: a step passes the drift of its products on several times over (against 64 bits, a stack
// of 256 x 1024: 4.7e-6 with 256, 2.9e-6 with 128, 1.8e-6 with 64; 4096 x 4096: 3.63, 3.84, 4.16 ms).
//
// p[]: [0..3] the product's (split: [0] partial sums of a matrix); [4] m, [5] n; [6] X to read, [7] X to write,
// [8] S, [9] P: byte offsets in scratch; [10] 1 when the step writes the float32 result.
#pragma once
#include "tcb/gemm_f16x3.cuh"

namespace tcb {

constexpr u32 NS_PARTS = 512;   // most partial sums of squares a matrix

struct Ns {
  const Args& a;
  __device__ explicit Ns(const Args& args) : a(args) {}
  __device__ u64 m() const { return (u64)a.p[4]; }
  __device__ u64 n() const { return (u64)a.p[5]; }
  __device__ double* parts() const { return reinterpret_cast<double*>(a.scratch); }
};

// 32 values of an fp16 pair array at (row, col), scaled by `down`.  Beyond the pitch the last 8 columns are
// read again (nothing uses those values): a branch around each load would have them wait one for another.
__device__ __forceinline__ void load_split32(float (&x)[32], const unsigned char* plane, u64 plane_bytes, u64 pitch,
                                             u64 row, u32 col, float down) {
  const unsigned char* p = plane + row * pitch * 2;
  uint4 hq[4], lq[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const u32 at = 2 * (col + 8 * c < (u32)pitch ? col + 8 * c : (u32)pitch - 8);
    hq[c] = *reinterpret_cast<const uint4*>(p + at);
    lq[c] = *reinterpret_cast<const uint4*>(p + plane_bytes + at);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 h = hq[c], l = lq[c];
    const u32 hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a, b, s, t;
      f16x2_float(hs[k], a, b);
      f16x2_float(ls[k], s, t);
      x[8 * c + 2 * k] = (a + s) * down;
      x[8 * c + 2 * k + 1] = (b + t) * down;
    }
  }
}

}  // namespace tcb

// Sums of squares in double (no float32 square can overflow it), a partial per block of a matrix.
extern "C" __global__ void __launch_bounds__(256) tcb_orth_norm(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  f16_clear(a, F16_CTRL);
  __shared__ double sh[8];
  const Ns s(a);
  const u64 count = s.m() * s.n();
  const float* x = reinterpret_cast<const float*>(a.in[0]) + (u64)blockIdx.y * count;
  double acc = 0.0;
  const u64 T = (u64)gridDim.x * 256, id = (u64)blockIdx.x * 256 + threadIdx.x;
  const u64 quads = (reinterpret_cast<u64>(x) & 15) == 0 ? count / 4 : 0;
#pragma unroll 4
  for (u64 i = id; i < quads; i += T) {
    const float4 q = __ldg(reinterpret_cast<const float4*>(x) + i);
    acc += (double)q.x * q.x + (double)q.y * q.y + ((double)q.z * q.z + (double)q.w * q.w);
  }
  for (u64 i = 4 * quads + id; i < count; i += T) acc += (double)ld1(x + i) * ld1(x + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 8; ++k) acc += sh[k];
    s.parts()[(u64)blockIdx.y * gridDim.x + blockIdx.x] = acc;
  }
}

// X = G / (|G|_F + eps) as hi and lo, row pitch n rounded up to 8.
extern "C" __global__ void __launch_bounds__(256) tcb_orth_split(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  const Ns s(a);
  const u64 m = s.m(), n = s.n(), pitch = (n + 7) / 8 * 8, b = blockIdx.y;
  __shared__ double sh[8];
  static_assert(NS_PARTS == 512, "a thread loads two partials");
  const u32 parts = (u32)a.p[0];
  const double* part = s.parts() + b * parts;
  double sum = (threadIdx.x < parts ? part[threadIdx.x] : 0.0) + (threadIdx.x + 256 < parts ? part[threadIdx.x + 256] : 0.0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += sh[k];
  const double inv = 1.0 / (sqrt(sum) + (double)(TCB_NS_EPS)) * (double)(1u << TCB_EX);
  const float* x = reinterpret_cast<const float*>(a.in[0]) + b * m * n;
  u32* out = reinterpret_cast<u32*>(a.scratch + (u64)a.p[6]) + b * m * pitch;
  const u64 plane = m * pitch / 2, segs = (n + 1023) / 1024;
  const bool wide = n % 4 == 0 && (reinterpret_cast<u64>(x) & 15) == 0;
  for (u64 u = blockIdx.x; u < m * segs; u += gridDim.x) {
    const u64 row = u / segs, c = (u % segs) * 1024 + 4 * threadIdx.x;
    if (c >= n) continue;
    float v[4];
    const float* r = x + row * n;
    if (wide) {
      load<4>(v, r + c);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c + j < n ? ld1(r + c + j) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)((double)v[j] * inv);
    uint2 hi, lo;
    split2(v[0], v[1], hi.x, lo.x);
    split2(v[2], v[3], hi.y, lo.y);
    u32* o = out + (row * pitch + c) / 2;
    *reinterpret_cast<uint2*>(o) = hi;
    *reinterpret_cast<uint2*>(o + plane) = lo;
  }
}

namespace tcb {

// S, or P = b S + c S S: written where computed and, when the tile across the diagonal is not computed,
// mirrored there.
template <int BN, int CTAS, bool POLY>
struct NsSymmetric {
  const Args& a;
  const TmaDesc* map;
  __device__ explicit NsSymmetric(const GemmParams& P) : a(P.a), map(&P.maps[2]) {}
  __device__ __forceinline__ void start(unsigned char*) {}
  __device__ __forceinline__ void begin(const F16Epi&) {}
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    const u64 M = (u32)a.p[0], pitch = (M + 7) / 8 * 8, plane = M * pitch * 2;   // bytes of a plane
    const u32 col = (u32)(e.T.n0 + c0);
    if (POLY) {
      float s[32];
      const u64 row = e.row < M ? e.row : M - 1;
      load_split32(s, reinterpret_cast<const unsigned char*>(a.scratch + (u64)a.p[8]) + (u64)e.T.bz * 2 * plane, plane,
                   pitch, row, col, pow2(TCB_EP - TCB_ES));
      const float up = pow2(TCB_EP - 2 * TCB_ES);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = fmaf(TCB_NS_C, v[j] * up, TCB_NS_B * s[j]);
    } else {
      const float up = pow2(TCB_ES - 2 * TCB_EX);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= up;
    }
    store_split32(e, map, v, (int)col, e.T.m0 + 32 * e.q, e.T.bz);
    const u32 row0 = (u32)e.T.m0 + 32 * e.q;
    if (row0 / BN < col / (CTAS * HG_M) * (CTAS * HG_M) / BN) {   // the mirror's tile is not computed
      if (e.lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      turn32(e, v);   // lane l: row l of the mirrored block
      store_split32(e, map, v, (int)row0, (int)col, e.T.bz);
    }
  }
  __device__ __forceinline__ void end(const F16Epi&) {}
  __device__ __forceinline__ void done(const F16Epi& e) {
    if (e.lane == 0) bulk_wait_all();
  }
};

// X = a X + P X (or X P): hi and lo for the next step, or the float32 result.
struct NsApply {
  const Args& a;
  const TmaDesc* map;
  __device__ explicit NsApply(const GemmParams& P) : a(P.a), map(&P.maps[2]) {}
  __device__ __forceinline__ void start(unsigned char*) {}
  __device__ __forceinline__ void begin(const F16Epi&) {}
  __device__ __forceinline__ void block(const F16Epi& e, int c0, float (&v)[32]) {
    const u64 m = (u64)a.p[4], n = (u64)a.p[5], pitch = (n + 7) / 8 * 8, plane = m * pitch * 2;
    const u32 col = (u32)(e.T.n0 + c0);
    const bool last = a.p[10] != 0;
    float x[32];
    load_split32(x, reinterpret_cast<const unsigned char*>(a.scratch + (u64)a.p[6]) + (u64)e.T.bz * 2 * plane, plane, pitch,
                 e.row < m ? e.row : m - 1, col, last ? pow2(-TCB_EX) : 1.0f);
    const float up = last ? pow2(-TCB_EP - TCB_EX) : pow2(-TCB_EP);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = fmaf(TCB_NS_A, x[j], v[j] * up);
    if (!last) {
      store_split32(e, map, v, (int)col, e.T.m0 + 32 * e.q, e.T.bz);
      return;
    }
    turn32(e, v);
    if (col + e.lane >= n) return;
    const u64 row0 = (u64)e.T.m0 + 32 * e.q;
    const int rows = (int)(m - row0 < 32 ? m - row0 : 32);
    float* o = reinterpret_cast<float*>(a.out) + ((u64)e.T.bz * m + row0) * n + col + e.lane;
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (r < rows) o[(u64)r * n] = v[r];
  }
  __device__ __forceinline__ void end(const F16Epi&) {}
  __device__ __forceinline__ void done(const F16Epi& e) {
    if (e.lane == 0) bulk_wait_all();
  }
};

}  // namespace tcb

#define TCB_NS_GEMM(NAME, TILE, BN, CTAS, AMN, BMN, SYM, EPI)                                                       \
  extern "C" __global__ void TCB_F16_CLUSTER_##CTAS __launch_bounds__(tcb::HG_THREADS, 1)                           \
      NAME##_##TILE(const __grid_constant__ tcb::GemmParams P) {                                                    \
    tcb::EPI epi(P);                                                                                                \
    tcb::gemm_f16x3<BN, CTAS, AMN, BMN, SYM, false, 128>(tcb::f16_job(P), reinterpret_cast<u32*>(P.a.p[15]), epi);  \
  }
#define TCB_NS_S(BN, CTAS) NsSymmetric<BN, CTAS, false>
#define TCB_NS_P(BN, CTAS) NsSymmetric<BN, CTAS, true>
// wide: X X^T (both along n), P X (X along n); tall: X^T X, X P (P = P^T); S S (S = S^T)
#define TCB_NS_GEMMS(TILE, BN, CTAS)                                                              \
  TCB_NS_GEMM(tcb_orth_gram_wide, TILE, BN, CTAS, false, false, true, TCB_NS_S(BN, CTAS))         \
  TCB_NS_GEMM(tcb_orth_gram_tall, TILE, BN, CTAS, true, true, true, TCB_NS_S(BN, CTAS))           \
  TCB_NS_GEMM(tcb_orth_poly, TILE, BN, CTAS, false, false, true, TCB_NS_P(BN, CTAS))              \
  TCB_NS_GEMM(tcb_orth_apply_wide, TILE, BN, CTAS, false, true, false, NsApply)                   \
  TCB_NS_GEMM(tcb_orth_apply_tall, TILE, BN, CTAS, false, false, false, NsApply)
TCB_F16_TILES(TCB_NS_GEMMS)
