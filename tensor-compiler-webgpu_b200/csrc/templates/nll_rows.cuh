// tcb/nll_rows.cuh -- the cross entropy of a few rows without a backward (scoring the next token of a handful of
// sequences): tcb/linear_nll.cuh's loss for at most 16 rows.
//
// Bound by reading W once.  The tensor core would need a pass for its largest magnitude, one that splits it and
// one that reads it back; here every value of W goes from memory into at most 16 float32 multiply-adds on the CUDA
// cores: 1 x 64 x 50001 34.6 -> 8.6 us, 4 x 276 x 89420 124 -> 25 us (W alone at the copy rate: 15), 16 x 1024 x
// 131072 464 -> 228 us (82), 16 x 64 x 65 12.3 -> 12.3 us.  Up to 4 rows W bounds it, at 16 the multiply-adds; with 32 the
// tensor core's form is ahead: 128 us against 166 at 1024 x 32000.
//
// A block takes 128 columns and a range of the d indices; lanes hold four columns each, warps take every eighth
// index, eight loads in flight, and h comes from shared memory four rows a load.  Each 32 columns of a row leave
// their maximum and sum of exponentials, which a block a row joins.  With few columns d is divided among blocks;
// tcb_nll_rows_add then adds the parts up, in order, first.
//
// p[]: [0] parts of d, [1] indices of a part, [2] byte offset in scratch of the targets' logits [R], [3] of the
// statistics [columns in 32s][R], [4] R, [5] d, [6] V; at 0 of scratch the parts' sums [parts][R][V], when there are
// several.  in[]: h, W, (b), t.
#pragma once
#include "tcb/nll_common.cuh"

namespace tcb {

constexpr int NR_K = 256;   // indices of h in shared memory at a time

// Where four rows of index k stand in its ROWS values: turned with k, so that the threads that write neighbouring
// indices meet in few banks.
template <int ROWS> __device__ __forceinline__ u32 nr_at(u32 g, u32 k) { return 4 * ((g + k) & (ROWS / 4 - 1)); }

// The maximum and the sum of exponentials of a warp's 32 columns of a row from a lane's sum, the target's logit.
__device__ __forceinline__ void nr_stats(const Args& a, u32 row, u64 c, float v) {
  const u64 R = (u64)a.p[4], V = (u64)a.p[6];
  const float b = TCB_BIAS ? ld1(reinterpret_cast<const float*>(a.in[2]) + (c < V ? c : V - 1)) : 0.0f;
  const int t = nll_class(ld1(reinterpret_cast<const float*>(a.in[TCB_BIAS ? 3 : 2]) + row), V);
  v = c < V ? fmaf(v, NLL_LOG2E, nll_bias2(b)) : TCB_MINUS_INF;
  if (t >= 0 && c == (u64)t) reinterpret_cast<float*>(a.scratch + (u64)a.p[2])[row] = v;
  const float m = warp_max(v);
  float s = ex2(v - (m == TCB_MINUS_INF ? 0.0f : m));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0 && c < V) reinterpret_cast<float2*>(a.scratch + (u64)a.p[3])[c / 32 * R + row] = make_float2(m, s);
}

template <int ROWS, bool WIDE>
__device__ __forceinline__ void nll_rows(const Args& a, float* sh) {   // sh: h, then 8 warps' 4 rows of 128 sums
  const u32 R = (u32)a.p[4];
  const u64 d = (u64)a.p[5], V = (u64)a.p[6];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const float* h = reinterpret_cast<const float*>(a.in[0]);
  const float* W = reinterpret_cast<const float*>(a.in[1]);
  const u64 c0 = (u64)blockIdx.x * 128, k0 = (u64)blockIdx.y * (u64)a.p[1];
  const u64 k1 = k0 + (u64)a.p[1] < d ? k0 + (u64)a.p[1] : d;
  // this lane's columns, the last one again beyond V (their sums are not written)
  u64 col[WIDE ? 1 : 4];
  if (WIDE) {
    col[0] = c0 + 4 * lane + 4 <= V ? c0 + 4 * lane : V - 4;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) col[WIDE ? 0 : j] = c0 + lane + 32 * j < V ? c0 + lane + 32 * j : V - 1;
  }
  float acc[ROWS][4];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[r][j] = 0.0f;
  for (u64 kc = k0; kc < k1; kc += NR_K) {
    const u32 n = (u32)(k1 - kc < NR_K ? k1 - kc : NR_K);
    __syncthreads();
    float y[ROWS];   // index threadIdx.x of every row (NR_K threads); beyond the rows the last again
    const u32 kh = threadIdx.x < n ? threadIdx.x : n - 1;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) y[r] = ld1(h + (r < R ? r : R - 1) * d + kc + kh);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) sh[threadIdx.x * ROWS + nr_at<ROWS>(r / 4, threadIdx.x) + r % 4] = threadIdx.x < n ? y[r] : 0.0f;
    __syncthreads();
    for (u32 kk = w; kk < n; kk += 64) {
      float x[8][4];
#pragma unroll
      for (int u = 0; u < 8; ++u) {   // beyond the part's end its last index again, for nothing
        const float* row = W + (kc + (kk + 8 * u < n ? kk + 8 * u : n - 1)) * V;
        if (WIDE) {
          load<4>(x[u], row + col[0]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[u][j] = ld1(row + col[WIDE ? 0 : j]);
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = kk + 8 * u < n ? x[u][j] : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {   // (left early the loop would have its loads wait one for another)
        const float* q = sh + (kk + 8 * u) * ROWS;
#pragma unroll
        for (int g = 0; g < ROWS / 4; ++g) {
          const float4 y = *reinterpret_cast<const float4*>(q + nr_at<ROWS>(g, kk + 8 * u));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[4 * g][j] = fmaf(y.x, x[u][j], acc[4 * g][j]);
            acc[4 * g + 1][j] = fmaf(y.y, x[u][j], acc[4 * g + 1][j]);
            acc[4 * g + 2][j] = fmaf(y.z, x[u][j], acc[4 * g + 2][j]);
            acc[4 * g + 3][j] = fmaf(y.w, x[u][j], acc[4 * g + 3][j]);
          }
        }
      }
    }
  }
  // the 8 warps' sums, four rows at a time, in order
  float* out = reinterpret_cast<float*>(a.scratch) + (u64)blockIdx.y * R * V;
#pragma unroll
  for (int g = 0; g < ROWS / 4; ++g) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) sh[(w * 4 + r) * 128 + (WIDE ? 4 * lane + j : lane + 32 * j)] = acc[4 * g + r][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32 r = (threadIdx.x + 256 * i) / 128, c = threadIdx.x % 128;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += sh[(k * 4 + r) * 128 + c];
      if (4 * g + r >= R) continue;
      if (gridDim.y == 1) nr_stats(a, 4 * g + r, c0 + c, v);
      else if (c0 + c < V) out[(4 * g + r) * V + c0 + c] = v;
    }
  }
}

}  // namespace tcb

#define TCB_NLL_ROWS(ROWS)                                                                        \
  extern "C" __global__ void __launch_bounds__(256) tcb_nll_rows_##ROWS(const tcb::Args a) {      \
    tcb::grid_dependency_sync();                                                                  \
    __shared__ __align__(16) float sh[tcb::NR_K * ROWS > 4096 ? tcb::NR_K * ROWS : 4096];         \
    if (a.p[6] % 4 == 0 && (a.in[1] & 15) == 0) tcb::nll_rows<ROWS, true>(a, sh);                 \
    else tcb::nll_rows<ROWS, false>(a, sh);                                                       \
  }
TCB_NLL_ROWS(4)
TCB_NLL_ROWS(8)
TCB_NLL_ROWS(16)

// The parts of d added up: a block a row and 256 columns.
extern "C" __global__ void __launch_bounds__(256) tcb_nll_rows_add(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  const u64 R = (u64)a.p[4], V = (u64)a.p[6], c = (u64)blockIdx.x * 256 + threadIdx.x;
  const float* part = reinterpret_cast<const float*>(a.scratch) + blockIdx.y * V + (c < V ? c : V - 1);
  float x[8], v = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = __ldcg(part + (k < (int)a.p[0] ? k : 0) * R * V);
#pragma unroll
  for (int k = 0; k < 8; ++k) v += k < (int)a.p[0] ? x[k] : 0.0f;
  nr_stats(a, blockIdx.y, c, v);
}

// A row's loss, a block a row.
extern "C" __global__ void __launch_bounds__(1024) tcb_nll_rows_finish(const tcb::Args a) {
  using namespace tcb;
  grid_dependency_sync();
  __shared__ float2 sh[32];
  const u64 R = (u64)a.p[4], V = (u64)a.p[6], row = blockIdx.x, n = (V + 31) / 32;
  const float2* p = reinterpret_cast<const float2*>(a.scratch + (u64)a.p[3]) + row;
  float m = TCB_MINUS_INF, s = 0.0f;
  for (u64 k = threadIdx.x; k < n; k += 4 * 1024) {
    float2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __ldcg(p + (k + 1024 * i < n ? k + 1024 * i : k) * R);
#pragma unroll
    for (int i = 0; i < 4; ++i) nll_join(m, s, k + 1024 * i < n ? x[i] : make_float2(TCB_MINUS_INF, 0.0f));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    nll_join(m, s, make_float2(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o)));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 1; k < 32; ++k) nll_join(m, s, sh[k]);
    const int t = nll_class(ld1(reinterpret_cast<const float*>(a.in[TCB_BIAS ? 3 : 2]) + row), V);
    const float z = __ldcg(reinterpret_cast<const float*>(a.scratch + (u64)a.p[2]) + row);
    reinterpret_cast<float*>(a.out)[row] = nll_loss(m, s, z, t, reinterpret_cast<const float*>(a.in[2]));
  }
}
